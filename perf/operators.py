"""The measured cases of three groups of operators, each in its plain form and as the framework's calls.

  product    8-bit matrix product with a scale per row of either operand ("token" and "channel"), float output; the rows
             of the left operand are either held in 8 bits already or quantised within the pass
               C[m, n] = (sum_k A[m, k] B[n, k]) sa[m] sb[n] + bias[n]
  topk       scores of 8-bit factor rows against an 8-bit item table with the k best items of every user kept
               score = RN(RN(RN(acc) sp) sq) + b, float32; order (score descending, id ascending); train items left out
  clip       global l2 norm over many gradient tensors, and every tensor scaled by max_norm / max(norm, max_norm)

An 8-bit row is q = nearest integer (ties to even) to x / scale with scale = max |x| / 127 in float32.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the smallest call: one user's scores over a catalogue of 1682 items, 20 factors (conf/BPR.ini on ML-100k)
        {"name": "product_one_user", "op": "product", "M": 1, "N": 1682, "K": 20, "x": "i8", "out": "f32", "bias": True},
        # one token through a square layer whose weights stay in 8 bits; bound by reading them
        {"name": "product_one_token", "op": "product", "M": 1, "N": 4096, "K": 4096, "x": "bf16", "out": "bf16", "bias": False},
        # a ragged batch of tokens, nothing a multiple of a tile
        {"name": "product_ragged", "op": "product", "M": 77, "N": 5003, "K": 1210, "x": "f32", "out": "f32", "bias": True},
        # a block of users against 200k items (the catalogue of the benchmark), all scores wanted: bound by writing them
        {"name": "product_all_scores", "op": "product", "M": 2048, "N": 200000, "K": 64, "x": "i8", "out": "f32", "bias": True},
        # a prompt through a wide layer: bound by the matrix cores
        {"name": "product_prompt", "op": "product", "M": 4096, "N": 8192, "K": 8192, "x": "bf16", "out": "bf16", "bias": False},
        # serving one user: the best 50 of 200k items
        {"name": "topk_one_user", "op": "topk", "n": 1, "I": 200000, "d": 64, "k": 50, "train": 40},
        # the ML-100k evaluation: every user against 1682 items, 20 factors
        {"name": "topk_small_eval", "op": "topk", "n": 943, "I": 1682, "d": 20, "k": 50, "train": 85},
        # a serving batch over the large catalogue (2M items, 128 factors, top 100): bound by reading the item table
        {"name": "topk_serving", "op": "topk", "n": 33, "I": 2000000, "d": 128, "k": 100, "train": 20},
        # a block of the full evaluation of the benchmark's model: 200k items, 64 factors
        {"name": "topk_eval", "op": "topk", "n": 4096, "I": 200000, "d": 64, "k": 50, "train": 16},
        # the gradients of the ML-100k model (two tables and a bias vector)
        {"name": "clip_small_model", "op": "clip", "tensors": 3, "total": 54182, "dtype": "f32", "spread": 4.0, "clipped": True},
        # many ragged tensors in 16 bits, from one element up
        {"name": "clip_many", "op": "clip", "tensors": 600, "total": 20000003, "dtype": "bf16", "spread": 1e6, "clipped": True},
        # the gradients of the benchmark's model (1M users and 200k items, 64 factors), norm within the bound
        {"name": "clip_large_model", "op": "clip", "tensors": 3, "total": 77000000, "dtype": "f32", "spread": 400.0, "clipped": False},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["product", "product", "topk", "clip"])
    if op == "product":
        K = _spread(rng, 8, 8192)
        N = _spread(rng, 64, 200000)
        M = _spread(rng, 1, 4096)
        # no more products, and no larger an output or weight table, than the largest listed cases
        N = min(N, max(64, (1 << 28) // K))
        M = max(1, min(M, 4096 * 8192 * 8192 // (N * K), 2048 * 200000 // N))
        return {"op": op, "M": M, "N": N, "K": K, "x": rng.choice(["i8", "f32", "bf16", "f16"]), "out": rng.choice(["f32", "f32", "bf16", "f16"]),
                "bias": rng.random() < 0.5}
    if op == "topk":
        d = _spread(rng, 8, 256)
        I = _spread(rng, 300, 2000000)
        n = max(1, min(_spread(rng, 1, 4096), 4096 * 200000 // I, 4096 * 200000 * 64 // (I * d)))
        return {"op": op, "n": n, "I": I, "d": d, "k": rng.choice([1, 10, 20, 50, 100, 200]), "train": _spread(rng, 1, 100)}
    tensors = _spread(rng, 1, 600)
    return {"op": op, "tensors": tensors, "total": max(tensors, _spread(rng, 1000, 70000000)), "dtype": rng.choice(["f32", "bf16", "f16"]),
            "spread": rng.choice([1.0, 10.0, 400.0, 1e6]), "clipped": rng.random() < 0.7}


# --------------------------------------------------------------------------------------------------------------- inputs
def _padded(d):
    return (d + 15) // 16 * 16


def _to_i8(x):
    """8-bit rows in their storage (whole groups of 16 columns, the rest zero) and their scales."""
    a = x.abs().amax(1, keepdim=True).double()
    s = (a / 127.0).float()
    q = torch.where(s > 0, torch.round(x.double() / s.double()), torch.zeros((), dtype=torch.float64, device=x.device)).clamp(-127, 127)
    out = torch.zeros((x.shape[0], _padded(x.shape[1])), dtype=torch.int8, device=x.device)
    out[:, :x.shape[1]] = q.to(torch.int8)
    return out, s.reshape(-1)


def _rows_i8(n, d, g, low=0.2, high=2.0):
    """8-bit rows of normal factors, whose lengths differ from row to row as trained rows' do, made a few rows at a time."""
    out = torch.empty((n, _padded(d)), dtype=torch.int8, device="cuda")
    scale = torch.empty(n, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // d)
    for r in range(0, n, step):
        m = min(step, n - r)
        x = torch.randn((m, d), generator=g, device="cuda") * torch.empty((m, 1), device="cuda").uniform_(low, high, generator=g)
        out[r:r + m], scale[r:r + m] = _to_i8(x)
    return out, scale


def _sizes(case, seed):
    """The lengths of the gradient tensors: `spread` is the ratio of the largest weight to the smallest."""
    g = torch.Generator().manual_seed(977 + seed % 7)
    n = case["tensors"]
    w = torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * math.log(case["spread"])) if case["spread"] > 1 else torch.ones(n, dtype=torch.float64)
    s = (w / w.sum() * (case["total"] - n)).long() + 1
    s[int(torch.argmax(s))] += case["total"] - int(s.sum())
    return s.tolist()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    st = dict(case)
    if case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        st["Bq"], st["sb"] = _rows_i8(N, K, g)
        st["biasv"] = torch.randn(N, generator=g, device="cuda") if case["bias"] else None
        if case["x"] == "i8":
            st["Aq"], st["sa"] = _rows_i8(M, K, g)
        else:
            st["X"] = torch.randn((M, K), generator=g, device="cuda").to(DTYPES[case["x"]])
            st["Aq"] = torch.zeros((M, _padded(K)), dtype=torch.int8, device="cuda")
            st["sa"] = torch.zeros(M, device="cuda")
        st["C"] = torch.zeros((M, N), dtype=DTYPES[case["out"]], device="cuda")
    elif case["op"] == "topk":
        n, I, d, k = case["n"], case["I"], case["d"], case["k"]
        st["Pq"], st["sp"] = _rows_i8(n, d, g)
        st["Qq"], st["sq"] = _rows_i8(I, d, g)
        st["b"] = torch.randn(I, generator=g, device="cuda")
        st["users"] = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
        most = max(1, min(2 * case["train"], I // 2))
        deg = torch.randint(0, most + 1, (n,), generator=g, device="cuda")
        ids = torch.randint(1, I // most + 1, (n, most), generator=g, device="cuda").cumsum(1) - 1
        st["train"] = (torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), deg.cumsum(0)]),
                       ids[torch.arange(most, device="cuda")[None, :] < deg[:, None]].to(torch.int32))
        st["ids"] = torch.zeros((n, k), dtype=torch.int32, device="cuda")
        st["scores"] = torch.zeros((n, k), device="cuda")
    else:
        sizes = _sizes(case, seed)
        total = sum(sizes)
        t = DTYPES[case["dtype"]]
        flat = (torch.randn(total, generator=g, device="cuda") * 0.01).to(t)
        st["flat"], st["out_flat"] = flat, torch.zeros_like(flat)
        st["grads"], st["outs"] = list(torch.split(flat, sizes)), list(torch.split(st["out_flat"], sizes))
        st["max_norm"] = 0.01 * math.sqrt(total) * (0.3 if case["clipped"] else 3.0)
        st["norm"] = torch.zeros(1, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------------------ one pass
_handle = {}


def _device():
    """The program's handle of the GPU, made once, on torch's current stream."""
    if "dev" not in _handle:
        from tfrec_amd.sharded import make_device
        _handle["dev"] = make_device(torch.cuda.current_device())
    return _handle["dev"]


def run(st):
    return {"product": _product, "topk": _topk, "clip": _clip}[st["op"]](st)


def _handles(st):
    """What a program makes once for its buffers and tables: the descriptions of 8-bit matrices, the list of gradients."""
    if "handles" not in st:
        from tfrec_amd.device import QuantRows
        if st["op"] == "product":
            st["handles"] = QuantRows(st["Aq"], st["sa"], st["K"]), QuantRows(st["Bq"], st["sb"], st["K"])
        elif st["op"] == "topk":
            st["handles"] = QuantRows(st["Pq"], st["sp"], st["d"]), QuantRows(st["Qq"], st["sq"], st["d"])
        else:
            st["handles"] = _device().grad_list(st["grads"], out=st["outs"])
    return st["handles"]


def _product(st):
    if own:
        dev, (a, b) = _device(), _handles(st)
        if st["x"] != "i8":
            dev.quantize_rows(st["X"], out=a)
        return {"C": dev.matmul_i8(a, b, bias=st["biasv"], out=st["C"])}
    K = st["K"]
    if st["x"] == "i8":
        a, sa = st["Aq"][:, :K].float(), st["sa"]
    else:
        x = st["X"].double()
        sa = (x.abs().amax(1) / 127.0).float()
        a = torch.where(sa[:, None] > 0, torch.round(x / sa[:, None].double()), torch.zeros((), dtype=torch.float64, device=x.device)).clamp(-127, 127).float()
    c = torch.matmul(a, st["Bq"][:, :K].float().t()) * sa[:, None] * st["sb"][None, :]
    if st["biasv"] is not None:
        c = c + st["biasv"][None, :]
    return {"C": c.to(DTYPES[st["out"]])}


def _topk(st):
    if own:
        p, q = _handles(st)
        ids, scores = _device().score_topk_i8(p, q, st["b"], st["users"], st["k"], train=st["train"], out_ids=st["ids"], out_scores=st["scores"])
        return {"ids": ids, "scores": scores}
    d, k, I = st["d"], st["k"], st["I"]
    users = st["users"].long()
    s = torch.matmul(st["Pq"][users][:, :d].float(), st["Qq"][:, :d].float().t())      # whole numbers below 2^24: exact
    s = s * st["sp"][users][:, None] * st["sq"][None, :] + st["b"][None, :]
    indptr, indices = st["train"]
    rows = torch.empty_like(users)
    rows[users] = torch.arange(len(users), device=s.device)
    s[torch.repeat_interleave(rows, indptr[1:] - indptr[:-1]), indices.long()] = -math.inf
    # (score, id) in one whole number: larger = ranks earlier
    bits = s.view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7fffffff)).long() * (1 << 32) + (I - 1 - torch.arange(I, device=s.device))[None, :]
    at = I - 1 - (torch.topk(key, min(k, I), dim=1).values & 0xffffffff)
    top = torch.gather(s, 1, at)
    at = torch.where(top == -math.inf, torch.full_like(at, -1), at)
    if k > I:
        at, top = torch.nn.functional.pad(at, (0, k - I), value=-1), torch.nn.functional.pad(top, (0, k - I), value=-math.inf)
    return {"ids": at.to(torch.int32), "scores": top}


def _clip(st):
    if own:
        _device().clip_grads(_handles(st), st["max_norm"], norm=st["norm"])
        return {"grads": st["out_flat"], "norm": st["norm"]}
    norm = torch.stack([x.double().square().sum() for x in st["grads"]]).sum().sqrt()
    scale = (st["max_norm"] / torch.clamp(norm, min=st["max_norm"])).float()
    return {"grads": torch.cat([(x.float() * scale).to(x.dtype) for x in st["grads"]]), "norm": norm.float().reshape(1)}


# --------------------------------------------------------------------------------------------- what a pass has to do
def work(case):
    if case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        x = M * K * SIZE[case["x"]] if case["x"] != "i8" else M * K + 4 * M
        return {"bytes": x + N * K + 4 * N + M * N * SIZE[case["out"]] + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    if case["op"] == "topk":
        n, I, d, k = case["n"], case["I"], case["d"], case["k"]
        return {"bytes": n * (d + 4) + I * (d + 8) + 4 * n + 4 * n * case["train"] + 8 * n * k, "flops": 2 * n * I * d}
    return {"bytes": 2 * case["total"] * SIZE[case["dtype"]] + 4, "flops": 3 * case["total"]}


# ------------------------------------------------------------------------------------------- the definition in 64 bits
def _nearest(x):
    """Rows in double precision -> (the whole numbers that an 8-bit row holds, its scale), row by row as defined."""
    top = torch.max(torch.max(x, 1).values, -torch.min(x, 1).values)
    scale = torch.div(top, torch.full_like(top, 127.0)).to(torch.float32).to(torch.float64)
    v = x * torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))[:, None]
    low = torch.floor(v)
    twice = 2.0 * (x - low * scale[:, None])                # against the scale: below the middle, on it, above it
    up = (twice > scale[:, None]) | ((twice == scale[:, None]) & (torch.remainder(low, 2.0) == 1.0))
    return torch.clamp(low + up.to(torch.float64), -127.0, 127.0), scale


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "product":
        K = case["K"]
        if case["x"] == "i8":
            a = st["Aq"][:, :K].to(torch.float64) * st["sa"].to(torch.float64)[:, None]
        else:
            q, scale = _nearest(st["X"].to(torch.float64))
            a = q * scale[:, None]
        del st["C"]
        c = torch.mm(a, (st["Bq"][:, :K].to(torch.float64) * st["sb"].to(torch.float64)[:, None]).t())
        return {"C": c if st["biasv"] is None else c.add_(st["biasv"].to(torch.float64))}
    if case["op"] == "topk":
        d, I, k = case["d"], case["I"], case["k"]
        u = st["users"].long()
        p = st["Pq"][:, :d].to(torch.float64) * st["sp"].to(torch.float64)[:, None]
        q = st["Qq"][:, :d].to(torch.float64) * st["sq"].to(torch.float64)[:, None]
        s = torch.addmm(st["b"].to(torch.float64)[None, :], p, q.t())             # in the order of the table's users
        indptr, indices = st["train"]
        lens = torch.diff(indptr)
        s.index_put_((torch.arange(len(lens), device=s.device).repeat_interleave(lens), indices.long()), torch.full((), -math.inf, dtype=torch.float64, device=s.device))
        best = torch.sort(torch.topk(s, min(k, I), dim=1).values, dim=1, descending=True).values[u]
        if k > I:
            best = torch.cat([best, torch.full((len(u), k - I), -math.inf, dtype=torch.float64, device=s.device)], 1)
        return {"ids": None, "scores": best}              # which of two scores one rounding apart comes first has no value in 64 bits
    x = st["flat"].to(torch.float64)
    norm = torch.linalg.vector_norm(x)
    return {"grads": x * (st["max_norm"] / max(float(norm), st["max_norm"])), "norm": norm.reshape(1)}
