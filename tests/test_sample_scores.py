"""``ops.sample_scores`` against a row-by-row oracle in 64 bits (numpy, python sums).

An answer is an index: it has to be equal.  The inputs are drawn so that no ``u * total`` lies
within 1e-10 of a step of the running weight and no top-p target within 1e-10 of one either (the
oracle says how near it came, both sides' sums are good to about 1e-12); such a draw
would say nothing about which side is right.  Where the steps are exact in both (equal
scores), the borders themselves are tested.
"""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from flink_parameter_server_1_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
INF = float("inf")


def oracle_row(s, u, T=1.0, k=0, p=1.0, q=0.0):
    """(index, probability, how near the answer is to another one)"""
    s = np.asarray(s, dtype=np.float64)
    live = np.flatnonzero(s > -INF)
    if live.size == 0:
        return -1, 0.0, 1.0
    v = s[live]
    best = v.max()
    if not T > 0:
        return int(live[np.argmax(v)]), 1.0, 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp(np.where(v == best, 0.0, (v - best) / T))
    rank = np.argsort(-v, kind="stable")
    if k > 0:
        rank = rank[:k]
    near = 1.0
    if p < 1:
        cum = np.cumsum(w[rank].astype(np.longdouble))
        before = np.concatenate([[0], cum[:-1]])
        target = p * cum[-1]
        near = min(near, float(np.abs(before[1:] - target).min() / cum[-1])) if rank.size > 1 else near
        rank = rank[: max(1, int((before < target).sum()))]
    if q > 0:
        rank = rank[w[rank] >= min(q, 1.0)]
    rank = np.sort(rank)
    cum = np.cumsum(w[rank].astype(np.longdouble))
    target = u * cum[-1]
    near = min(near, float(np.abs(cum - target).min() / cum[-1]))
    hit = min(int(np.searchsorted(cum, target, side="right")), rank.size - 1)
    while w[rank[hit]] == 0:
        hit -= 1
    return int(live[rank[hit]]), float(w[rank[hit]] / cum[-1]), near


def check(S, u, dev, near_ok=False, **kw):
    """Runs the op, compares with the oracle; settings are numbers or per-row lists."""
    B = S.shape[0]
    args, rows = {}, {}
    for key, short in (("temperature", "T"), ("top_k", "k"), ("top_p", "p"), ("min_p", "q")):
        if key in kw:
            v = kw[key]
            if isinstance(v, (list, tuple)):
                t = torch.tensor(v, dtype=torch.int32 if key == "top_k" else torch.float32)
                args[key], rows[short] = t.to(dev), t.double().tolist()
            else:
                args[key], rows[short] = v, [v] * B
    idx, prob = ops.sample_scores(S.to(dev), u.to(dev), with_prob=True, **args)
    assert idx.dtype == torch.int32 and prob.dtype == torch.float32
    s = S.double().numpy()
    for b in range(B):
        opts = {key: (int(v[b]) if key == "k" else v[b]) for key, v in rows.items()}
        want, pr, near = oracle_row(s[b], float(u[b]), **opts)
        assert near_ok or near > 1e-10, "choose another seed"
        assert int(idx[b]) == want, (b, int(idx[b]), want, opts)
        assert abs(float(prob[b]) - pr) <= 2.0**-23 * pr, (b, float(prob[b]), pr)
    again = ops.sample_scores(S.to(dev), u.to(dev), **args)
    assert torch.equal(again, idx)
    return idx


def scores(B, n, seed, spread=3.0, masked=0.1, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    s = torch.randn(B, n, generator=g) * spread
    if masked:
        s[torch.rand(B, n, generator=g) < masked] = -INF
    return s.to(dtype), torch.rand(B, generator=g)


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=5), dict(top_k=40, top_p=0.9),
            dict(top_p=0.5), dict(top_p=0.95, temperature=1.5), dict(min_p=0.1), dict(top_k=700, top_p=0.99),
            dict(top_k=20, top_p=0.8, min_p=0.05, temperature=0.5), dict(top_p=0.9, min_p=0.3), dict(temperature=0.0),
            dict(temperature=50.0, top_p=0.7), dict(temperature=0.01, top_k=30), dict(top_k=10**9), dict(top_p=0.0),
            dict(top_k=9000), dict(top_k=9000, top_p=0.97, min_p=0.001), dict(top_k=15000, top_p=0.3), dict(min_p=1e-4),
            dict(top_k=9000, min_p=0.02, temperature=2.0), dict(top_k=300, top_p=0.5, temperature=30.0)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [1, 2, 63, 256, 257, 1000, 4096, 4097, 32768, 32769, 70001])
@pytest.mark.parametrize("case", range(len(SETTINGS)))
def test_against_the_oracle(dev, n, case):
    S, u = scores(3, n, seed=1000 * case + n)
    check(S, u, dev, **SETTINGS[case])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [50, 5000, 40000])
@pytest.mark.parametrize("case", [0, 4, 5, 6, 8, 9, 11, 12])
def test_16_bit_scores_with_their_ties(dev, dtype, n, case):
    S, u = scores(3, n, seed=77 * case + n, dtype=dtype)
    check(S, u, dev, **SETTINGS[case])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [300, 6000, 50000])
def test_settings_per_row(dev, n):
    B = 12
    S, u = scores(B, n, seed=n)
    S[5] = -INF
    check(S, u, dev, temperature=[1, 0, 0.5, 2, 1, 1, -1, 1, 0.1, 30, 1, 1],
          top_k=[0, 3, 10, 0, n, 4, 9, -2, 600, 0, 1, 100], top_p=[1, 0.5, 0.9, 0.8, 0.99, 0.5, 0.5, 2, 0.7, 0.6, 0.9, 0.0],
          min_p=[0, 0, 0.1, 0, 0.01, 0.5, 0, -1, 0, 0.2, 0, 5.0])
    check(S, u, dev, top_k=[n // 2, 0, 700, n // 3, 5, 0, n // 2, 2000, 0, 900, 4000, n - 1],
          top_p=[0.9, 0.9, 1, 0.2, 0.9, 0.3, 1, 0.999, 1, 0.7, 0.0, 0.95], min_p=[0, 0, 0, 0, 0, 0, 0.01, 0, 0.2, 0.1, 0, 0])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [8, 1000, 5000, 40000, 200000])
def test_equal_scores_go_by_index(dev, n):
    """Every weight is 1: borders are whole numbers, exact on every side."""
    S = torch.full((6, n), 2.5)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0**-24, 0.125])
    check(S, u, dev, near_ok=True)
    k = n // 2
    i = check(S, u, dev, near_ok=True, top_k=k)
    assert int(i.max()) < k
    i = check(S, u, dev, near_ok=True, top_p=0.25)
    assert int(i.max()) < n // 4  # n is a multiple of 4: the border itself is cut
    i = check(S, u, dev, near_ok=True, top_k=n - n // 4, top_p=0.5)
    assert int(i.max()) < (n - n // 4) // 2
    check(S, u, dev, near_ok=True, top_k=k, top_p=0.5, min_p=1.0)
    S[:, ::2] = 1.0
    # top-k takes all of the better half and some ties, top-p ends above them, among them, at them
    for p in (0.25, 0.5, 0.75, 0.875):
        check(S, u, dev, near_ok=True, top_k=n // 2 + n // 8, top_p=p, temperature=1e9)
    check(S, u, dev, near_ok=True, temperature=0.0)
    check(S, u, dev, near_ok=True, top_k=3)
    S[:] = 0.0
    S[:, 1::2] = -0.0  # one score
    check(S, u, dev, near_ok=True, top_k=5)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [10, 3000, 9000, 36000])
def test_masks_infinities_and_nan(dev, n):
    S, u = scores(9, n, seed=3 * n, masked=0)
    S[0] = -INF
    S[1] = float("nan")
    S[2] = -INF
    S[2, n - 1] = -7.0
    S[3, ::2] = float("nan")
    S[4, [1, n // 2, n - 1]] = INF
    S[5, 3] = INF
    S[6] = torch.finfo(torch.float32).min  # a mask by the lowest value: everything equal
    S[7, 1:] = torch.finfo(torch.float32).min
    S[8] = -INF
    S[8, 2] = torch.finfo(torch.float32).min
    for kw in (dict(), dict(top_k=2), dict(top_p=0.6), dict(top_k=4, top_p=0.5, min_p=0.01), dict(temperature=0.0),
               dict(min_p=0.5), dict(top_k=n - 1, top_p=0.9), dict(top_k=n // 2, top_p=0.7), dict(top_k=n // 2)):
        check(S, u, dev, near_ok=True, **kw)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [100, 3000, 9000, 40000])
def test_temperatures_next_to_zero(dev, n):
    """Only the best score has weight, every one of those equal to it alike (zero takes the first)."""
    S, u = scores(4, n, seed=n)
    S[1, [3, n // 2, n - 1]] = 99.0
    S[2, [1, n - 2]] = INF
    for kw in (dict(), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.5), dict(top_k=n // 2), dict(top_k=n // 2, top_p=0.9)):
        for T in (1e-310, 5e-324, 1e-45, [2.0**-149] * 4):
            i = check(S, u, dev, near_ok=True, temperature=T, **kw)
            if not kw and T == 1e-310:
                assert int(i[1]) in (3, n // 2, n - 1) and int(i[2]) in (1, n - 2)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(SETTINGS)))
def test_rows_past_a_million(case):
    """More segments than a workgroup keeps in LDS (4096 of 256 scores)."""
    S, u = scores(2, 1_200_003, seed=31 * case + 1)
    check(S, u, "cuda", **SETTINGS[case])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(top_k=600_000), dict(top_p=0.25), dict(top_k=900_000, top_p=0.5),
                                dict(top_k=5), dict(min_p=1.0), dict(top_k=600_000, top_p=0.5, min_p=1.0)])
def test_a_million_equal_scores(kw):
    S, u = torch.full((3, 1_200_000), -4.0), torch.tensor([0.0, 0.62501, 1 - 2.0**-24])
    check(S, u, "cuda", near_ok=True, **kw)
    S[1] = S[1].bfloat16()
    S[1, ::3] = -5.0  # two scores; the last row's all but one masked
    S[2, 1:] = -INF
    check(S, u, "cuda", near_ok=True, **dict(kw, temperature=1e9))


@pytest.mark.gpu
def test_16_bit_rows_past_a_million():
    """Few different values: bins hold more scores than a list, ties by the thousand."""
    S, u = scores(2, 1_200_003, seed=2, dtype=torch.bfloat16)
    for kw in (dict(top_k=500_000), dict(top_p=0.5), dict(top_k=500_000, top_p=0.9), dict(top_p=0.9, temperature=40.0)):
        check(S, u, "cuda", **kw)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A score matrix of more than 2^31 entries and 2^32 bytes; its last row against the same row alone."""
    B, n = 66, 33_000_000
    S = torch.empty(B, n, dtype=torch.bfloat16, device="cuda")
    S[:-1] = float("-inf")
    S[-1] = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    u = torch.full((B,), 0.7, device="cuda")
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.2)):
        i = ops.sample_scores(S, u, **kw)
        alone = ops.sample_scores(S[-1:], u[-1:], **kw)
        assert bool((i[:-1] == -1).all()) and int(i[-1]) == int(alone[0]) >= 0


@pytest.mark.gpu
def test_more_rows_than_a_launch_takes():
    B = (1 << 22) + 70
    S = torch.randn(B, 3, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    u = torch.rand(B, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    k = (torch.arange(B, device="cuda") % 4).int()
    T, p, q = (torch.full((B,), v, device="cuda") for v in (0.8, 0.9, 0.05))
    idx, prob = ops.sample_scores(S, u, temperature=T, top_k=k, top_p=p, min_p=q, with_prob=True)
    for a, b in ((0, 1000), ((1 << 22) - 500, B)):
        i, r = ops.sample_scores(S[a:b].cpu(), u[a:b].cpu(), temperature=T[a:b].cpu(), top_k=k[a:b].cpu(),
                                 top_p=p[a:b].cpu(), min_p=q[a:b].cpu(), with_prob=True)
        assert torch.equal(idx[a:b].cpu(), i) and torch.allclose(prob[a:b].cpu(), r, rtol=2.0**-22, atol=0)
    assert bool((idx >= 0).all()) and bool((idx < 3).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_u_at_and_outside_its_range(dev):
    S, _ = scores(4, 1000, seed=5, masked=0)
    S[:, 0] = S[:, -1] = -INF
    i = ops.sample_scores(S.to(dev), torch.tensor([0.0, -1.0, 1.0, float("nan")], device=dev))
    assert i.tolist() == [1, 1, 998, 998]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [100, 5000, 40000])
def test_strided_rows(dev, n):
    """A column slice of a wider score matrix: rows off 16 bytes, others' scores around it."""
    big = torch.full((5, n + 9), 50.0)
    S, u = scores(5, n, seed=9)
    for first in (0, 3, 4):
        big[:] = 50.0
        big[:, first:first + n] = S
        view = big.to(dev)[:, first:first + n]
        for kw in (dict(), dict(top_k=7, top_p=0.9), dict(top_p=0.8)):
            assert torch.equal(ops.sample_scores(view, u.to(dev), **kw), ops.sample_scores(S.to(dev), u.to(dev), **kw))


@pytest.mark.parametrize("dev", DEVICES)
def test_draws_follow_the_weights(dev):
    """4096 evenly spaced u on one row: every index as often as its weight says, within one."""
    S, _ = scores(1, 200, seed=12, spread=1.0)
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    i = ops.sample_scores(S.expand(n, 200).contiguous().to(dev), u.to(dev), temperature=0.8)
    p = torch.softmax(S[0].double() / 0.8, 0)
    count = torch.bincount(i.cpu().long(), minlength=200).double()
    assert float((count - n * p).abs().max()) <= 1.0 + 1e-6


@pytest.mark.parametrize("dev", DEVICES)
def test_empty(dev):
    assert ops.sample_scores(torch.empty(0, 5, device=dev), torch.empty(0, device=dev)).shape == (0,)
    i, p = ops.sample_scores(torch.empty(3, 0, device=dev), torch.empty(3, device=dev), with_prob=True)
    assert i.tolist() == [-1, -1, -1] and not p.any()


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    S, u = torch.zeros(3, 10, device=dev), torch.zeros(3, device=dev)
    bad = [dict(S=S[0]), dict(S=S.double()), dict(S=S.t().contiguous().t()), dict(S=S[:1].expand(3, 10)),
           dict(u=u[:2]), dict(u=u.double()), dict(temperature=-0.5), dict(temperature=float("nan")),
           dict(temperature=INF), dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=1.1),
           dict(min_p=float("nan")), dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:2]),
           dict(min_p=torch.zeros(6, device=dev)[::2])]
    for kw in bad:
        kw = dict(dict(S=S, u=u), **kw)
        with pytest.raises(ValueError):
            ops.sample_scores(kw.pop("S"), kw.pop("u"), **kw)


@pytest.mark.gpu
def test_two_devices_are_refused():
    S = torch.zeros(3, 10, device="cuda")
    with pytest.raises(ValueError):
        ops.sample_scores(S, torch.zeros(3))
    with pytest.raises(ValueError):
        ops.sample_scores(S, torch.zeros(3, device="cuda"), top_p=torch.ones(3))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3000, 60000])
def test_replayed_draws_equal_eager_ones(n):
    S, u = (t.cuda() for t in scores(6, n, seed=4))
    p = torch.full((6,), 0.9, device="cuda")
    call = lambda: (ops.sample_scores(S, u, top_k=40, top_p=p), ops.sample_scores(S, u, top_p=p),  # noqa: E731
                    ops.sample_scores(S, u, temperature=0.5))
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for k in range(4):
        a, b = scores(6, n, seed=50 + k)
        S.copy_(a)
        u.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, call()):
            assert torch.equal(x, y)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_two_streams_at_once():
    """Workspaces are per call: two streams drawing from different matrices do not meet."""
    data = [scores(8, 50000, seed=s) for s in (1, 2)]
    dev = [(a.cuda(), b.cuda()) for a, b in data]
    want = [ops.sample_scores(a, b, top_p=0.9) for a, b in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dev]
    got = [[], []]
    for _ in range(10):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[j].append(ops.sample_scores(*dev[j], top_p=0.9))
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(x, want[j]) for x in got[j])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [100, 3000, 9000, 40000])
def test_min_p_next_to_a_best_score_of_zero(dev, n):
    """Rows whose best score is zero or subnormal, at temperatures at which the least weight that min-p keeps lies
    no fp32 step below the best one: the best one stays, and it is what remains."""
    S, u = scores(6, n, seed=7 * n)
    S[0] = 0.0
    S[1].clamp_(max=0.0)                      # many best scores
    S[2] = -S[2].abs() - 0.5
    S[2, n // 3] = 0.0                        # one
    S[3] = -INF
    S[3, n - 2] = 0.0
    S[4] = 1e-40
    S[5] = S[5].clamp(max=0.0) - 1e-40
    for T in (1e-310, 5e-324, 1e-46, [2.0**-149] * 6):
        for q in (0.9, 0.05, 1.0, [0.5] * 6):
            for kw in (dict(), dict(top_k=n // 2 + 1), dict(top_k=n // 2 + 1, top_p=0.7), dict(top_p=0.7), dict(top_k=3)):
                check(S, u, dev, near_ok=True, temperature=T, min_p=q, **kw)


def flat_tail(n, B, tail_mass, seed):
    """Rows of one best score over equal ones, which hold `tail_mass` of its weight together."""
    g = torch.Generator().manual_seed(seed)
    S = torch.full((B, n), float(np.log(tail_mass / (n - 1))))
    S[torch.arange(B), torch.randint(0, n, (B,), generator=g)] = 0.0
    S[0] = S[0, 1]
    S[0, 0] = 0.0
    return S


def tail_row(n, best, w, u, top_k=0, top_p=1.0, min_p=0.0):
    """(index, probability, distance to a step in steps) in whole and rational numbers: ``n - 1`` scores of weight ``w`` (all
    above ``min_p``) around one of weight 1.  (A running sum loses it: n roundings at 2^-64 are a tenth of a step.)"""
    w, u, kept = Fraction(w), Fraction(u), (top_k or n) - 1
    off = Fraction(1, 2)
    if top_p < 1:
        border = (Fraction(top_p) * (1 + kept * w) - 1) / w  # tie number j stays while j < border
        off = min(off, abs(border - round(border)))
        kept = min(kept, max(0, math.ceil(border)))
    total = 1 + kept * w
    target, before = u * total, min(best, kept)
    if target < before * w or target >= before * w + 1:
        x = target / w if target < before * w else (target - 1) / w
        m = min(math.floor(x), kept - 1)
        return m + (m >= best), float(w / total), float(min(off, abs(x - round(x))))
    return best, float(1 / total), float(min(off, (target - before * w) / w, (before * w + 1 - target) / w))


def check_tail(n, dev, tail_mass, B=4):
    """The draws that fall into the tail.  A step there is far below 1e-10 of the total, and still one index: the sums
    have to be right to a hundredth of it."""
    S = flat_tail(n, B, tail_mass, seed=n)
    k = n - n // 10
    w = float(np.exp(np.float64(S[0, 1])))
    p, pk = ((1 + (int(0.6 * kept) + 0.5) * w) / (1 + (kept - 1) * w) for kept in (n, k))  # half way between two steps
    for kw in (dict(), dict(top_k=k), dict(min_p=1e-30), dict(top_p=p), dict(top_k=k, top_p=pk), dict(top_k=k, min_p=1e-30),
               dict(top_k=400, min_p=1e-30), dict(top_k=k, top_p=pk, min_p=1e-30)):
        tried = 0
        for part in (0.13, 0.29, 0.37, 0.49, 0.52, 0.58):
            u = torch.full((B,), float(1 - part * tail_mass / (1 + tail_mass)))
            idx, prob = ops.sample_scores(S.to(dev), u.to(dev), with_prob=True, **kw)
            for b in range(B):
                want, pr, near = tail_row(n, int(S[b].argmax()), w, float(u[b]), **kw)
                if near < 0.01:
                    continue  # next to a step
                tried += 1
                assert int(idx[b]) == want, (b, int(idx[b]), want, near, kw)
                assert abs(float(prob[b]) - pr) <= 2.0**-23 * pr, (b, float(prob[b]), pr, kw)
        assert tried >= 1


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [1000, 9000, 16000, 40000, 70001])
@pytest.mark.parametrize("tail_mass", [0.3, 2.0**-14, 2.0**-19])
def test_a_best_score_over_a_flat_tail(dev, n, tail_mass):
    check_tail(n, dev, tail_mass)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1_000_000, 1_200_003])
@pytest.mark.parametrize("tail_mass", [0.3, 1.4e-5, 2.0**-21])
def test_a_best_score_over_a_long_flat_tail(n, tail_mass):
    check_tail(n, "cuda", tail_mass)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,p_best", [(25, 0.99977), (28, 0.985)])
def test_the_tail_of_very_long_rows(bits, p_best):
    """One best score, the others together 1 - p_best: their number times a weight far below 2^-31."""
    n = 1 << bits
    tail = torch.tensor(np.log((1 / p_best - 1) / n)).bfloat16()
    S = torch.empty(1, n, dtype=torch.bfloat16, device="cuda")
    S[:] = tail
    S[0, 0] = 0
    w = float(np.exp(np.float64(tail.float())))
    for kw, kept in ((dict(top_k=n // 2), n // 2), (dict(min_p=1e-12), n), (dict(), n),
                     (dict(top_k=n // 2, min_p=1e-12), n // 2)):
        total = 1 + (kept - 1) * w
        i, p = ops.sample_scores(S, torch.tensor([0.5], device="cuda"), with_prob=True, **kw)
        assert int(i[0]) == 0 and abs(float(p[0]) - 1 / total) <= 2.0**-23
        u = float(torch.tensor(1 - 0.3 * (total - 1) / total).float())
        i, p = ops.sample_scores(S, torch.tensor([u], device="cuda"), with_prob=True, **kw)
        # weights are good to 1.1e-12 each, sums to 2^-61 for each segment of 256
        assert abs(int(i[0]) - ((u * total - 1) / w + 1)) <= 1.5
        assert abs(float(p[0]) * total / w - 1) <= 2.0**-23


def check_ends(n, dev):
    """u at and outside the ends of its range: the first and the last kept score, however small their weights are."""
    g = torch.Generator().manual_seed(n)
    u = torch.tensor([0.0, -1.0, 1.0, float("nan"), 1 - 2.0**-24, 2.0])
    S = -30 - 50 * torch.rand(6, n, generator=g)
    S[torch.arange(6), torch.randint(n // 4, n // 2, (6,), generator=g)] = 0.0
    for kw in (dict(), dict(top_k=2), dict(top_k=40), dict(top_k=200), dict(top_k=n // 2), dict(top_k=n - 1),
               dict(min_p=1e-30), dict(top_k=40, min_p=1e-25), dict(top_k=n // 2, min_p=1e-25)):
        check(S, u, dev, near_ok=True, **kw)
    S += 3.0  # nor does the best score's own value matter
    check(S, u, dev, near_ok=True, top_k=n // 2)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [50, 300, 2000, 9000, 40000])
def test_ends_of_rows_of_tiny_weights(dev, n):
    check_ends(n, dev)


@pytest.mark.gpu
def test_ends_of_long_rows_of_tiny_weights():
    check_ends(1_200_003, "cuda")


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [3000, 40000])
def test_scores_apart_by_more_than_the_type_holds(dev, n):
    """Differences past fp32's range that a temperature past it makes small again."""
    S, u = scores(4, n, seed=n + 1, masked=0.1)
    S = S.clamp(-8, 8) * 4e37
    S[1] = -3e38
    S[1, ::256] = 3e38  # one score of each 256
    S[2] = torch.finfo(torch.float32).min
    S[2, ::300] = 1.0
    for T in (1e39, 3e38, 1e300, [3e38] * 4):
        for kw in (dict(), dict(top_p=0.61), dict(top_k=n // 2, top_p=0.61), dict(min_p=0.2), dict(top_p=0.61, min_p=0.2)):
            check(S, u, dev, near_ok=True, temperature=T, **kw)


def test_row_counts_past_32_bits_are_refused():
    """(tensors without memory: nothing but their shapes is looked at)"""
    for B, n in ((2**31 + 5, 1), (2**32 + 3, 2), (3, 2**31)):
        with pytest.raises(ValueError):
            ops.sample_scores(torch.empty(B, n, device="meta"), torch.empty(B, device="meta"))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("n", [2047, 2048, 2049, 16383, 16384, 16385])
@pytest.mark.parametrize("case", range(len(SETTINGS)))
def test_lengths_at_which_the_path_changes(dev, n, case):
    """A segment per wave in registers up to 2048 scores, one launch without a workspace up to 16384."""
    S, u = scores(2, n, seed=5000 * case + n)
    check(S, u, dev, **SETTINGS[case])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1_048_576, 1_048_577])
@pytest.mark.parametrize("case", [0, 4, 5, 7, 17, 18, 20])
def test_lengths_at_which_maxima_leave_lds(n, case):
    S, u = scores(1, n, seed=6000 * case + n)
    check(S, u, "cuda", **SETTINGS[case])


def test_workspace_by_length_and_settings():
    from flink_parameter_server_1_amd.ops import _native
    from flink_parameter_server_1_amd.ops.sample import _SHORT_ROW

    if not _native.available():
        pytest.skip("kernel library not built")

    def size(B, n, T=1.0, k=0, p=1.0, q=0.0):
        return _native.require().fps_sample_scores_ws_bytes(B, n, None, T, None, k, None, p, None, q)

    assert size(5, _SHORT_ROW, p=0.5) == 0 < size(5, _SHORT_ROW + 1)
    n, segments = 131072, 512
    for kw in (dict(), dict(T=0.0, p=0.5, q=0.5), dict(k=100, p=0.9, q=0.1), dict(k=n), dict(T=0.0, k=5000)):
        assert size(256, n, **kw) <= 256 * segments * 16 + 16  # a maximum, a mass, a count per segment
    for kw in (dict(p=0.9), dict(q=0.1), dict(k=5000), dict(k=n, p=0.9)):
        assert size(256, n, **kw) > 256 * 16384 * 16


@pytest.mark.gpu
@pytest.mark.parametrize("n,dtype", [(1500, torch.float32), (60000, torch.float32), (60000, torch.bfloat16),
                                     (1_200_003, torch.float32)])
def test_draws_do_not_depend_on_the_order_of_atomics(n, dtype):
    """The same call again and again, and captured and replayed: indices and probabilities to the last bit."""
    S, u = (t.cuda() for t in scores(8, n, seed=n, spread=1.0, dtype=dtype))
    k = torch.tensor([0, 40, 600, n // 2, n // 3, 0, 7, n - 1], dtype=torch.int32, device="cuda")
    p = torch.tensor([0.9, 0.8, 1.0, 0.95, 1.0, 1.0, 0.5, 0.99], device="cuda")
    q = torch.tensor([0.0, 0.0, 0.01, 0.001, 0.0, 0.02, 0.0, 0.0], device="cuda")
    call = lambda: ops.sample_scores(S, u, top_k=k, top_p=p, min_p=q, with_prob=True)  # noqa: E731
    i, r = call()
    for _ in range(20):
        j, s = call()
        assert torch.equal(i, j) and torch.equal(r, s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        j, s = call()
    for _ in range(3):
        j.fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(i, j) and torch.equal(r, s)
        call()
        torch.cuda.synchronize()
