"""The microscaled-table and sampling operators, as measured work.

Four operators that serve answers from an item table:

* ``ops.mx_set_rows`` / ``ops.mx_gather_rows`` (cases ``table-*``): rows of a table held in
  4 or 8 bits per value, in blocks of 32 with one power-of-two scale, written by index and
  read back;
* ``ops.mx_score`` (``score-*``): inner products of queries with every row of such a table;
* ``ops.sample_scores`` (``sample-*``): one index per row of scores, drawn with temperature,
  top-k, top-p and min-p from given uniform numbers, and the probability it was drawn with.

``run`` is one pass through an operator: with ``own`` false in elementary torch operations,
with ``own`` true by the framework's calls.
"""
import numpy as np
import torch

own = False

BLOCK = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EMAX = {"fp4": 2, "fp8": 8}
BITS = {"fp4": 4, "fp8": 8}


def listed():
    return [
        # one updated item row put into a small index and the index read back: latency
        _table("table-fp8-one-row", slots=257, n=1, dim=64, fmt="fp8", src="fp32", out="fp32"),
        # a micro-batch of updated item rows (rank 64) into a serving index, read for a rebuild
        _table("table-fp4-batch-d64", slots=65536, n=4096, dim=64, fmt="fp4", src="bf16", out="bf16"),
        # word vectors of 300 values: ragged last block, a fifth of the vocabulary rewritten
        _table("table-fp8-words-d300", slots=100003, n=20011, dim=300, fmt="fp8", src="fp32", out="fp32"),
        # the whole item side of the rank-64 factorisation (1M items) written and read
        _table("table-fp4-all-items-d64", slots=1000000, n=1000000, dim=64, fmt="fp4", src="fp32", out="fp32"),
        # one user against 1M items of rank 64: the single-query answer
        _score("score-fp4-one-query-d64", b=1, n=1000000, dim=64, q="bf16", x="fp4", out="fp32"),
        # a few queries against word vectors held in 8 bits, odd sizes
        _score("score-fp8-words-d300", b=37, n=100003, dim=300, q="bf16", x="fp8", out="fp32"),
        # a query batch against the items, scores kept in bf16 for the sampler
        _score("score-fp4-batch-d64", b=256, n=1000000, dim=64, q="bf16", x="fp4", out="bf16"),
        # wide rows, both sides in 4 bits: bound by the product
        _score("score-fp4-fp4-wide-d4096", b=512, n=65536, dim=4096, q="fp4", x="fp4", out="bf16"),
        # one answer from a small catalogue
        _sample("sample-one-row-1k", b=1, n=1000, src="fp32", temperature=0.8, top_k=40, top_p=0.95, min_p=0.0),
        # a batch of users over all items, a short list and its nucleus
        _sample("sample-topk-1m", b=32, n=1000000, src="fp32", temperature=0.7, top_k=100, top_p=0.9, min_p=0.02),
        # nucleus alone over a large vocabulary, each row with its own settings
        _sample("sample-topp-128k-rows", b=128, n=131072, src="bf16", temperature=1.0, top_k=0, top_p=0.9,
                min_p=0.0, per_row=True),
        # the untruncated softmax over all items
        _sample("sample-softmax-1m", b=16, n=1000000, src="fp32", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
    ]


def _table(name, **kw):
    return dict(name=name, op="table", **kw)


def _score(name, **kw):
    return dict(name=name, op="score", **kw)


def _sample(name, per_row=False, **kw):
    return dict(name=name, op="sample", per_row=per_row, **kw)


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["table", "score", "sample"])
    if op == "table":
        dim = rng.choice([_log_int(rng, 1, 1024), 64, 128, 300])
        slots = _log_int(rng, 64, min(1000000, 64000000 // dim))
        return dict(op=op, slots=slots, n=_log_int(rng, 1, slots), dim=dim, fmt=rng.choice(["fp4", "fp8"]),
                    src=rng.choice(["fp32", "bf16", "fp16"]), out=rng.choice(["fp32", "bf16", "fp16"]))
    if op == "score":
        q, x = rng.choice([("bf16", "fp4"), ("bf16", "fp8"), ("fp4", "fp4")])
        dim = rng.choice([_log_int(rng, 8, 4096), 64, 128, 300])
        b = rng.choice([1, _log_int(rng, 1, 512)])
        n = _log_int(rng, 1000, min(1000000, 268000000 // dim, 256000000 // b))
        return dict(op=op, b=b, n=n, dim=dim, q=q, x=x, out=rng.choice(["fp32", "bf16", "fp16"]))
    b = _log_int(rng, 1, 256)
    n = _log_int(rng, 100, min(1000000, 33000000 // b))
    return dict(op=op, b=b, n=n, src=rng.choice(["fp32", "bf16", "fp16"]), temperature=rng.choice([0.0, 0.5, 0.8, 1.0, 1.5]),
                top_k=rng.choice([0, 1, 20, 100, _log_int(rng, 1, n)]), top_p=rng.choice([1.0, 0.5, 0.9, 0.95]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), per_row=rng.random() < 0.5)


def _padded(dim):
    return (dim + BLOCK - 1) // BLOCK * BLOCK


def _packed_bytes(rows, dim, fmt):
    return rows * (_padded(dim) * BITS[fmt] // 8 + _padded(dim) // BLOCK)


def _random_table(gen, rows, dim, fmt):
    """A packed table as earlier writes left it: codes of normally distributed rows,
    scales of a few octaves, zeros behind the last value of a row."""
    P = _padded(dim)
    x = torch.randn(rows, P, generator=gen, device="cuda")
    x[:, dim:] = 0
    # lengths of rows differ as item popularity does
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device="cuda"))
    data, scale = _encode(x, fmt)
    return dict(data=data, scale=scale)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = dict(case=case)
    if case["op"] == "table":
        T, n, D = case["slots"], case["n"], case["dim"]
        st["table"] = _random_table(gen, T, D, case["fmt"])
        x = torch.randn(n, D, generator=gen, device="cuda") * torch.exp(torch.randn(n, 1, generator=gen, device="cuda"))
        st["rows"] = x.to(TYPES[case["src"]])
        # distinct slots, as a micro-batch without repeats has them; every 17th row is padding
        idx = torch.randperm(T, generator=gen, device="cuda")[:n].to(torch.int32)
        if n > 16:
            idx[16::17] = -1
        st["idx"] = idx
        # the read visits every slot, in another order, and some padding
        read = torch.randperm(T, generator=gen, device="cuda").to(torch.int32)
        st["read"] = torch.cat([read, torch.full((3,), -1, dtype=torch.int32, device="cuda")])
        handles = ["table"]
    elif case["op"] == "score":
        st["q"] = (torch.randn(case["b"], case["dim"], generator=gen, device="cuda") * 0.3).bfloat16()
        st["x"] = _random_table(gen, case["n"], case["dim"], case["x"])
        handles = ["x"]
    else:
        B, N = case["b"], case["n"]
        # scores of a trained model: a normal bulk with a heavier upper tail, rows of different
        # sharpness; one item in 50 is excluded, in every 16th row nearly everything
        s = torch.randn(B, N, generator=gen, device="cuda")
        s = s * (1 + 1.5 * torch.rand(B, 1, generator=gen, device="cuda")) + 0.15 * s.clamp_min(0) ** 2
        gone = torch.rand(B, N, generator=gen, device="cuda")
        limit = torch.full((B, 1), 0.02, device="cuda")
        limit[15::16] = 0.999
        st["s"] = s.masked_fill_(gone < limit, float("-inf")).to(TYPES[case["src"]])
        st["u"] = torch.rand(B, generator=gen, device="cuda")
        for key in ("temperature", "top_k", "top_p", "min_p"):
            v = case[key]
            if case["per_row"]:
                if key == "top_k":
                    v = torch.full((B,), v, dtype=torch.int32, device="cuda")
                    v[3::4] = min(50, case["n"])
                else:
                    v = torch.full((B,), v, dtype=torch.float32, device="cuda")
                    if key == "temperature":
                        v[1::2] *= 0.75
                    if key == "top_p":
                        v[2::5] = 0.75
                    if key == "min_p":
                        v[4::7] = 0.05
            st[key] = v
        handles = []
    if own:
        from flink_parameter_server_1_amd import ops

        for h in handles:
            t = st[h]
            st[h + "_handle"] = ops.MXTable.wrap(t["data"], t["scale"], case["dim"], case["fmt"] if h == "table" else case["x"])
    return st


def run(state):
    case = state["case"]
    if own:
        from flink_parameter_server_1_amd import ops

        if case["op"] == "table":
            ops.mx_set_rows(state["table_handle"], state["idx"], state["rows"])
            return ops.mx_gather_rows(state["table_handle"], state["read"], out_dtype=TYPES[case["out"]])
        if case["op"] == "score":
            q = state["q"] if case["q"] == "bf16" else ops.MXTable.from_rows(state["q"], "fp4")
            return ops.mx_score(q, state["x_handle"], out_dtype=TYPES[case["out"]])
        return ops.sample_scores(state["s"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                                 top_p=state["top_p"], min_p=state["min_p"], with_prob=True)
    if case["op"] == "table":
        return _plain_table(state, case)
    if case["op"] == "score":
        return _plain_score(state, case)
    return _plain_sample(state)


# ---- the plain forms ---------------------------------------------------------------------


def _power(e):
    """2^e in fp32 for whole e in [-127, 127], exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64).float()


def _encode(x, fmt):
    """Codes and scale bytes of float rows whose width is a multiple of the block."""
    n, P = x.shape
    v = x.float().view(n, P // BLOCK, BLOCK)
    amax = v.abs().amax(2)
    scale = ((amax.view(torch.int32) >> 23) - EMAX[fmt]).clamp(0, 254)
    scale = torch.where(torch.isfinite(amax), scale, torch.full_like(scale, 255))
    y = v * _power(127 - scale.clamp_max(254))[:, :, None]
    if fmt == "fp8":
        code = y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        code = torch.where((scale == 255)[:, :, None], torch.zeros_like(code), code)
        return code.reshape(n, P), scale.to(torch.uint8)
    a = y.abs()
    # the number of midpoints passed; a midpoint itself goes to the even code
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int())
    code = (code + 8 * torch.signbit(y).int()) * (scale != 255)[:, :, None]
    code = code.reshape(n, P // 2, 2)
    return (code[:, :, 0] + 16 * code[:, :, 1]).to(torch.uint8), scale.to(torch.uint8)


def _decode(data, scale, dim, fmt):
    n = data.shape[0]
    if fmt == "fp8":
        v = data.view(torch.float8_e4m3fn).float()
    else:
        lut = torch.tensor(E2M1 + tuple(-e for e in E2M1), device=data.device)
        b = data.int()
        v = torch.stack([lut[b & 15], lut[b >> 4]], 2).reshape(n, -1)
    e = scale.int()
    f = _power(e.clamp_max(254) - 127)
    f = torch.where(e == 255, torch.full_like(f, float("nan")), f)
    return (v.view(n, -1, BLOCK) * f[:, :, None]).reshape(n, -1)[:, :dim]


def _pad(x):
    return torch.nn.functional.pad(x, (0, _padded(x.shape[1]) - x.shape[1]))


def _plain_table(state, case):
    dim, fmt = case["dim"], case["fmt"]
    values = _decode(state["table"]["data"], state["table"]["scale"], dim, fmt)
    new = _decode(*_encode(_pad(state["rows"]), fmt), dim, fmt)
    idx = state["idx"].long()
    live = idx >= 0
    values[idx[live]] = new[live]
    read = state["read"].long()
    out = values[read.clamp_min(0)] * (read >= 0)[:, None]
    return out.to(TYPES[case["out"]])


def _plain_score(state, case):
    q = state["q"].float()
    if case["q"] == "fp4":
        q = _decode(*_encode(_pad(q), "fp4"), case["dim"], "fp4")
    x = _decode(state["x"]["data"], state["x"]["scale"], case["dim"], case["x"])
    return (q @ x.t()).to(TYPES[case["out"]])


def _column(v, like):
    if not torch.is_tensor(v):
        v = torch.full((like.shape[0],), v, dtype=torch.float64, device=like.device)
    return v.double()[:, None]


def _plain_sample(state):
    s, u = state["s"].float(), state["u"].double()[:, None]
    B, N = s.shape
    T, k = _column(state["temperature"], s), _column(state["top_k"], s)
    p, min_p = _column(state["top_p"], s), _column(state["min_p"], s)
    s = torch.where(torch.isnan(s), torch.full_like(s, float("-inf")), s)
    # descending, equal scores in the order of their index
    ss, order = torch.sort(s, dim=1, descending=True, stable=True)
    top = ss[:, :1]
    z = torch.where(ss == top, torch.zeros_like(ss, dtype=torch.float64),
                    (ss.double() - top.double()) / T.clamp_min(1e-300))
    w = torch.where(ss == float("-inf"), torch.zeros_like(z), torch.exp(z))
    rank = torch.arange(N, device=s.device)[None, :]
    w = w * ((rank < k) | (k <= 0)) * ((rank < 1) | (T > 0))
    mass = torch.cumsum(w, 1)
    keep = ((mass - w < p * mass[:, -1:]) | (p >= 1) | (rank < 1)) & (w >= min_p)
    w = torch.zeros_like(w).scatter_(1, order, w * keep)
    mass = torch.cumsum(w, 1)
    total = mass[:, -1:]
    passed = (mass > u * total) & (w > 0)
    pos = torch.arange(N, device=s.device, dtype=torch.int32)[None, :].expand(B, N)
    first = torch.where(passed, pos, torch.full_like(pos, N)).amin(1)
    last = torch.where(w > 0, pos, torch.full_like(pos, -1)).amax(1)
    index = torch.where(first < N, first, last)
    drawn = torch.gather(w, 1, index.clamp_min(0).long()[:, None]) / total
    return index, torch.where(index >= 0, drawn[:, 0], torch.zeros_like(drawn[:, 0])).float()


def work(case):
    if case["op"] == "table":
        es_in, es_out = (2 if case["src"] != "fp32" else 4), (2 if case["out"] != "fp32" else 4)
        n, T, D = case["n"], case["slots"], case["dim"]
        byte = n * D * es_in + 4 * n + _packed_bytes(n, D, case["fmt"])          # write
        byte += 4 * T + _packed_bytes(T, D, case["fmt"]) + T * D * es_out        # read
        return {"bytes": byte, "flops": 2 * (n + T) * D}
    if case["op"] == "score":
        es = 2 if case["out"] != "fp32" else 4
        byte = _packed_bytes(case["n"], case["dim"], case["x"]) + 2 * case["b"] * case["dim"]
        return {"bytes": byte + es * case["b"] * case["n"], "flops": 2 * case["b"] * case["n"] * case["dim"]}
    es = 2 if case["src"] != "fp32" else 4
    return {"bytes": case["b"] * case["n"] * es + 12 * case["b"], "flops": 4 * case["b"] * case["n"]}


# ---- the operators' definitions in 64 bits -----------------------------------------------


def _two_to(e):
    """2^e in 64 bits for whole e in [-300, 300), from a table."""
    return torch.tensor([2.0**k for k in range(-300, 300)], dtype=torch.float64, device=e.device)[e.long() + 300]


def _exact_blocks(x, fmt):
    """Values that rows ``x`` (float64, width a multiple of the block) stand for once held
    in ``fmt``: every element on the grid of its own binade, ties to even."""
    v = x.view(x.shape[0], -1, BLOCK)
    amax = v.abs().amax(2, keepdim=True)
    _, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1)
    e = torch.where(amax > 0, (e - 1 - EMAX[fmt]).clamp(-127, 127), torch.full_like(e, -127))
    unit = _two_to(e)
    y = v / unit
    lowest, digits, largest = (0, 1, 6.0) if fmt == "fp4" else (-6, 3, 448.0)
    _, b = torch.frexp(y)
    b = torch.where(y == 0, torch.full_like(b, lowest + 1), b)
    step = _two_to((b - 1).clamp_min(lowest) - digits)
    y = (torch.round(y / step) * step).clamp(-largest, largest)
    return (y * unit).reshape(x.shape[0], -1)


def _exact_unpack(t, dim, fmt):
    """Float64 values of a packed table, from the fields of its codes."""
    data, scale = t["data"].long(), t["scale"].long()
    if fmt == "fp4":
        code = torch.stack([data % 16, data // 16], 2).reshape(data.shape[0], -1)
        sign, e, m, digits, bias = code // 8, code // 2 % 4, code % 2, 1, 1
    else:
        sign, e, m, digits, bias = data // 128, data // 8 % 16, data % 8, 3, 7
    frac = m.double() / 2**digits
    v = torch.where(e > 0, (1 + frac) * _two_to(e - bias), frac * 2.0 ** (1 - bias))
    v = torch.where(sign > 0, -v, v).view(data.shape[0], -1, BLOCK) * _two_to(scale - 127)[:, :, None]
    return v.reshape(data.shape[0], -1)[:, :dim]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "table":
        dim, fmt = case["dim"], case["fmt"]
        values = _exact_unpack(st["table"], dim, fmt)
        new = _exact_blocks(_pad(st["rows"].double()), fmt)[:, :dim]
        idx, read = st["idx"].long(), st["read"].long()
        values.index_copy_(0, idx[idx >= 0], new[idx >= 0])
        return torch.where(read[:, None] >= 0, values[read.clamp_min(0)], torch.zeros((), dtype=torch.float64, device="cuda"))
    if case["op"] == "score":
        q = st["q"].double()
        if case["q"] == "fp4":
            q = _exact_blocks(_pad(q), "fp4")[:, :case["dim"]]
        return q @ _exact_unpack(st["x"], case["dim"], case["x"]).t()
    if case["b"] * case["n"] > 40000000:
        return None
    B = case["b"]
    s, u = st["s"].double().cpu().numpy(), st["u"].double().cpu().numpy()
    par = {}
    for key in ("temperature", "top_k", "top_p", "min_p"):
        v = st[key]
        par[key] = v.double().cpu().numpy() if torch.is_tensor(v) else np.full(B, float(v))
    out, prob = np.full(B, -1, dtype=np.int32), np.zeros(B)
    for b in range(B):
        live = np.flatnonzero(s[b] > -np.inf)  # NaN is not larger either
        if live.size == 0:
            continue
        val = s[b][live]
        best = val.max()
        if par["temperature"][b] <= 0:
            out[b], prob[b] = live[np.argmax(val)], 1.0
            continue
        with np.errstate(invalid="ignore"):
            w = np.exp(np.where(val == best, 0.0, (val - best) / par["temperature"][b]))
        rank = np.argsort(-val, kind="stable")
        k = int(par["top_k"][b])
        if k > 0:
            rank = rank[:k]
        if par["top_p"][b] < 1:
            before = np.concatenate([[0.0], np.cumsum(w[rank])])
            rank = rank[: max(1, int(np.sum(before[:-1] < par["top_p"][b] * before[-1])))]
        rank = np.sort(rank[w[rank] >= par["min_p"][b]])
        mass = np.cumsum(w[rank])
        hit = np.searchsorted(mass, u[b] * mass[-1], side="right")
        hit = min(hit, rank.size - 1)
        out[b], prob[b] = live[rank[hit]], w[rank[hit]] / mass[-1]
    return torch.from_numpy(out).cuda(), torch.from_numpy(prob).cuda()
