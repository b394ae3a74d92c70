"""What the 4-bit operators of the engine are measured on: quantisation of rows to microscaled 4-bit numbers ("mx4"), the
product of queries with mx4 rows, the top-k search over an mx4 index, and the lookup of stored rows by id.

mx4: 32 consecutive elements of a row share one scale 2^s, s = floor(log2(largest magnitude)) - 2 (not below -127); an
element is the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times the scale, ties to the even code, magnitudes beyond 6 to 6.
The last block of a row may be short.

Every case says in a comment what it stands for. `own` is set from outside: False computes the plain forms in torch, True
calls the engine.
"""
import math

import torch

own = False

BLOCK = 32
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FLT_MAX = torch.finfo(torch.float32).max


def listed():
    return [
        # one query vector, quantised and read back: nothing but latency
        {"name": "quantize one vector", "op": "quantize", "n": 1, "d": 768, "type": "f32"},
        # an encoder's half-precision shard of passage vectors on its way into 4 bits
        {"name": "quantize a shard", "op": "quantize", "n": 500_000, "d": 768, "type": "f16"},
        # one query against a whole small corpus: bound by the rows it streams
        {"name": "scores of one query", "op": "scores", "nq": 1, "n": 100_000, "d": 768, "type": "f32"},
        # the small evaluation set, full score matrix (distillation targets, threshold studies)
        {"name": "scores of an evaluation set", "op": "scores", "nq": 1000, "n": 100_000, "d": 768, "type": "f32"},
        # short vectors, odd sizes, half-precision queries
        {"name": "scores odd", "op": "scores", "nq": 333, "n": 50_021, "d": 100, "type": "bf16"},
        # near-duplicate check of a block of stored 4-bit rows against others: both sides in mx4
        {"name": "scores of 4-bit rows", "op": "scores", "nq": 8192, "n": 32_768, "d": 768, "type": "mx4"},
        # a handful of queries on a toy corpus: launches and one round trip
        {"name": "search tiny", "op": "search", "nq": 3, "n": 999, "d": 100, "k": 10},
        # one interactive query on a passage corpus
        {"name": "search one query", "op": "search", "nq": 1, "n": 1_800_000, "d": 768, "k": 100},
        # a serving batch on the same corpus
        {"name": "search a batch", "op": "search", "nq": 64, "n": 1_800_000, "d": 768, "k": 100},
        # an evaluation run at the command's default depth
        {"name": "search an evaluation set", "op": "search", "nq": 1000, "n": 500_000, "d": 768, "k": 1000},
        # the passages of one result list, weighted by their scores
        {"name": "lookup one list", "op": "lookup", "n": 100_000, "d": 768, "m": 100, "type": "f32"},
        # the passages of an evaluation run's lists, for a re-ranker that reads bf16
        {"name": "lookup many lists", "op": "lookup", "n": 1_800_000, "d": 768, "m": 698_000, "type": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _dim(rng):
    """Vector lengths: any from 17 to 1536, the common multiples of 32 half the time."""
    d = _log_uniform(rng, 17, 1536)
    return d if rng.random() < 0.5 else max(32, d // 32 * 32)


def draw(rng):
    op = rng.choice(["quantize", "scores", "search", "lookup"])
    d = _dim(rng)
    if op == "quantize":
        return {"op": op, "n": _log_uniform(rng, 1, 500_000 * 768 // max(d, 768)), "d": d,
                "type": rng.choice(["f32", "f16", "bf16"])}
    if op == "scores":
        n = _log_uniform(rng, 1, 100_000)
        nq = _log_uniform(rng, 1, max(1, min(8192, 70_000_000 // n)))
        return {"op": op, "nq": nq, "n": n, "d": min(d, 1024), "type": rng.choice(["f32", "f16", "bf16", "mx4"])}
    if op == "search":
        n = _log_uniform(rng, 300, 1_200_000)
        nq = _log_uniform(rng, 1, max(1, min(1000, 100_000_000 // n)))
        return {"op": op, "nq": nq, "n": n, "d": min(d, 1024), "k": _log_uniform(rng, 1, 1000)}
    return {"op": op, "n": _log_uniform(rng, 1, 400_000), "d": d, "m": _log_uniform(rng, 1, 698_000 * 768 // max(d, 768) // 2),
            "type": rng.choice(["f32", "f16", "bf16"])}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(n, d, g):
    """Representations as encoders give them: unnormalised, some coordinates larger than others."""
    x = torch.randn(n, d, generator=g, device="cuda")
    x *= torch.exp(0.25 * torch.randn(n, 1, generator=g, device="cuda"))
    x *= torch.exp(0.25 * torch.randn(d, generator=g, device="cuda"))
    return x


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    g = _generator(seed)
    op, d = case["op"], case["d"]
    x = _rows(case["n"], d, g)
    if op == "quantize":
        return {"x": x.to(TYPES[case["type"]])}
    if op == "scores":
        q = _rows(case["nq"], d, g)
        return {"x": x, "q": q if case["type"] == "mx4" else q.to(TYPES[case["type"]])}
    if op == "search":
        # queries from an 8-bit encoder head: whole multiples of 1/32 (every score is then a number that 32 bits hold, so
        # that equal scores are equal in any order of summation and the order of the ids is defined)
        q = torch.randn(case["nq"], d, generator=g, device="cuda")
        return {"x": x, "q": torch.clamp(torch.round(q * 32), -127, 127) / 32}
    m = case["m"]
    ids = torch.randint(0, case["n"], (m,), generator=g, device="cuda")
    ids[torch.rand(m, generator=g, device="cuda") < 0.02] = -1          # empty slots of short result lists
    return {"x": x, "ids": ids, "scale": torch.rand(m, generator=g, device="cuda")}


def prepare(case, seed):
    t = _inputs(case, seed)
    op, d = case["op"], case["d"]
    state = {"op": op, "d": d, "k": case.get("k"), "type": case.get("type")}
    if op == "quantize":
        return {**state, **t}
    x = t.pop("x")
    state.update(t)
    if own:                     # the index a serving program builds once
        from mural_amd import mx4
        from mural_amd.faiss_retriever import FlatIPIndex
        state["index"] = FlatIPIndex(d, device=x.device.index, storage="mx4")
        state["index"].add(x)
        if case.get("type") == "mx4":
            state["q"] = mx4.quantize(state["q"])
    else:                       # the rows' values, kept in 32 bits
        state["rows"] = _quantized(x)
        if case.get("type") == "mx4":
            state["q"] = _quantized(state["q"])
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    op = s["op"]
    if op == "quantize":
        from mural_amd import mx4
        codes, scales = mx4.quantize(s["x"])
        return mx4.dequantize(codes, scales, s["d"])
    if op == "scores":
        return s["index"].scores_mx4(*s["q"]) if s["type"] == "mx4" else s["index"].scores(s["q"])
    if op == "search":
        return s["index"].search_device(s["q"], s["k"])
    return s["index"].lookup(s["ids"], s["scale"], dtype=TYPES[s["type"]])


def _quantized(x):
    """The values that the mx4 form of x [n, d] stands for, in 32 bits."""
    n, d = x.shape
    v = x.float()
    if d % BLOCK:
        v = torch.nn.functional.pad(v, (0, BLOCK - d % BLOCK))
    v = v.reshape(n, -1, BLOCK)
    largest = v.abs().amax(2, keepdim=True)
    _, e = torch.frexp(largest)                                           # largest = m 2^e, 0.5 <= m < 1
    e = torch.clamp(torch.where(largest > 0, e - 3, -127), min=-127)
    v = torch.ldexp(v, -e)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.clamp(torch.round(a / step) * step, max=6.0)                # torch.round: ties to even
    return torch.ldexp(torch.copysign(a, v), e).reshape(n, -1)[:, :d].contiguous()


def _run_plain(s):
    op = s["op"]
    if op == "quantize":
        return _quantized(s["x"])
    if op == "scores":
        return s["q"].float() @ s["rows"].T
    if op == "search":
        return _search(s["q"] @ s["rows"].T, s["k"])
    ids = s["ids"]
    rows = s["rows"][ids.clamp(min=0)] * (s["scale"] * (ids >= 0))[:, None]
    return rows.to(TYPES[s["type"]])


def _search(scores, k):
    """Top k of every row of scores (32 bits), equal scores by ascending column; (-FLT_MAX, -1) beyond the last column."""
    nq, n = scores.shape
    bits = scores.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64) << 32
    key += (1 << 32) - 1 - torch.arange(n, device=scores.device)
    ids = (1 << 32) - 1 - (torch.topk(key, min(k, n), dim=1).values & 0xFFFFFFFF)
    best = torch.gather(scores, 1, ids)
    if k > n:
        best = torch.nn.functional.pad(best, (0, k - n), value=-FLT_MAX)
        ids = torch.nn.functional.pad(ids, (0, k - n), value=-1)
    return best, ids


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    op, d, n = case["op"], case["d"], case["n"]
    row = 17 * -(-d // BLOCK)                                             # 16 bytes of codes and one of scale a block
    size = {"f32": 4, "f16": 2, "bf16": 2, "mx4": row / d}
    if op == "quantize":                                                  # rows in, 4 bits out and in again, values out
        return {"bytes": n * d * size[case["type"]] + 2 * n * row + 4 * n * d, "flops": 0}
    if op == "scores":
        nq = case["nq"]
        return {"bytes": n * row + nq * d * size[case["type"]] + 4 * nq * n, "flops": 2 * nq * n * d}
    if op == "search":
        nq = case["nq"]
        return {"bytes": n * row + 4 * nq * d + 12 * nq * case["k"], "flops": 2 * nq * n * d}
    m = case["m"]
    return {"bytes": min(m, n) * row + m * (12 + d * size[case["type"]]), "flops": m * d}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def _exact_quantized(x):
    """The mx4 values of x in 64 bits, block by block, by counting the midpoints that a magnitude lies beyond."""
    n, d = x.shape
    out = torch.empty(n, d, dtype=torch.float64, device=x.device)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    for j in range(0, d, BLOCK):
        v = x[:, j:j + BLOCK].double()
        top = v.abs().amax(1, keepdim=True)
        s = torch.floor(torch.log2(torch.clamp(top, min=2.0 ** -149)))
        s = torch.where(torch.exp2(s) > top, s - 1, s)                    # log2 rounds: at a power of two it may be one off
        s = torch.where(torch.exp2(s + 1) <= top, s + 1, s)
        s = torch.clamp(s - 2, min=-127)
        u = v.abs() / torch.exp2(s)
        # a tie goes to the even code: the upper one at 0.75, 1.75 and 3.5
        code = ((u > 0.25).long() + (u >= 0.75) + (u > 1.25) + (u >= 1.75) + (u > 2.5) + (u >= 3.5) + (u > 5.0))
        out[:, j:j + BLOCK] = torch.sign(v) * grid[code] * torch.exp2(s)
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    op = case["op"]
    x = _exact_quantized(t["x"])
    if op == "quantize":
        return x
    if op == "lookup":
        ids = t["ids"]
        out = x[torch.where(ids < 0, 0, ids)]
        out *= torch.where(ids < 0, 0.0, t["scale"].double())[:, None]
        return out
    q = _exact_quantized(t["q"]) if case.get("type") == "mx4" else t["q"].double()
    if op == "scores":
        return torch.matmul(q, x.t())
    n, k = case["n"], case["k"]
    best = torch.full((case["nq"], k), -FLT_MAX, dtype=torch.float64, device=x.device)
    rows = torch.full((case["nq"], k), -1, dtype=torch.int64, device=x.device)
    step = max(1, 200_000_000 // n)
    for i in range(0, case["nq"], step):
        s = torch.matmul(q[i:i + step], x.t())
        order = torch.sort(s, dim=1, descending=True, stable=True)        # stable: equal scores stay in row order
        best[i:i + step, :n] = order.values[:, :k]
        rows[i:i + step, :n] = order.indices[:, :k]
    return best, rows
