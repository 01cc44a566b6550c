"""qd_sample_rows: one token per row with per-row temperature, top-k, top-p, min-p and a given
random number, against the definition in 64 bits.

A drawn index may differ from the 64-bit one only where the border lies within the weights'
resolution: each of V weights is off by at most 2^-45 (half a step of 2^-44), so running sums by
V * 2^-45 in units of the largest weight; where the definition's own margin is below twice
that, the neighbouring token is accepted as well."""
import math

import numpy as np
import pytest

from kernel_optimization_webgpu_b200 import _lib


def test_arguments_are_refused():
    L = _lib.load()
    p = 4096
    assert L.qd_sample_rows(p, 1, -1, 10, 10, None, None, None, None, p, p, None, None) == _lib.QD_E_INVALID
    assert L.qd_sample_rows(p, 1, 1, 0, 10, None, None, None, None, p, p, None, None) == _lib.QD_E_INVALID
    assert L.qd_sample_rows(p, 5, 1, 10, 10, None, None, None, None, p, p, None, None) == _lib.QD_E_INVALID
    assert L.qd_sample_rows(p, 1, 2, 10, 9, None, None, None, None, p, p, None, None) == _lib.QD_E_INVALID
    assert L.qd_sample_rows(p, 1, 1, 393217, 393217, None, None, None, None, p, p, None, None) == _lib.QD_E_RANGE
    assert b"vocab" in L.qd_last_error(None)
    for logits, u, ids in ((None, p, p), (p, None, p), (p, p, None)):
        assert L.qd_sample_rows(logits, 1, 1, 10, 10, None, None, None, None, u, ids, None, None) == _lib.QD_E_INVALID
    assert L.qd_sample_rows(None, 1, 0, 10, 10, None, None, None, None, None, None, None, None) == _lib.QD_OK


def test_python_wrapper_refuses():
    torch = pytest.importorskip("torch")
    from kernel_optimization_webgpu_b200 import runtime as R
    x, u = torch.zeros(2, 9), torch.zeros(2)
    for args, kw in (((x[0], u), {}), ((x, u[:1]), {}), ((x, u.double()), {}), ((x.t(), u), {}), ((x.long(), u), {}),
                     ((x, u), dict(top_k=u)), ((x, u), dict(temperature=u[:1])), ((x, u), {})):
        with pytest.raises(ValueError):
            R.sample_rows(*args, **kw)


def definition(v, T, k, top_p, min_p, u):
    """(accepted ids, logprob of the first) in 64 bits; v: float64 values of one row."""
    V = v.size
    key = np.where(np.isnan(v), -np.inf, v)
    order = np.lexsort((np.arange(V), np.isnan(v), -key))
    best = v[order[0]]
    if not T > 0 or k == 1 or not np.isfinite(best):
        return [int(order[0])], 0.0
    n = k if 0 < k < V else V
    with np.errstate(over="ignore", invalid="ignore"):
        w = np.where(np.isnan(v[order]), 0.0, np.exp((key[order] - best) / T))[:n]
    unit = V * 2.0 ** -44
    run = np.cumsum(w)
    cuts = [w.size]
    if top_p < 1:
        goal = max(top_p, 0.0) * run[-1]
        cuts = sorted({min(int((run < g).sum()) + 1, w.size) for g in (goal - unit, goal, goal + unit)})
        mid = min(int((run < goal).sum()) + 1, w.size)
    else:
        mid = w.size
    few = int((w >= min_p).sum()) if min_p > 0 else w.size
    accepted, logp = [], None
    for m in [mid] + cuts:
        m = max(1, min(m, few))
        live = m if w[m - 1] > 0 else int((w[:m] > 0).sum())
        for g in (u * run[m - 1], u * run[m - 1] - unit, u * run[m - 1] + unit):
            i = min(int((run[:m] <= max(g, 0.0)).sum()), live - 1)
            if logp is None:
                logp = math.log(w[i] / run[m - 1])
            accepted.append(int(order[i]))
    return accepted, logp


def _cuda():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def check(torch, x, T, k, p, mp, u):
    from kernel_optimization_webgpu_b200 import runtime as R
    f = lambda a: torch.tensor(a, dtype=torch.float32, device="cuda")  # noqa: E731
    ids, logp = R.sample_rows(x, f(u), temperature=f(T), top_k=torch.tensor(k, dtype=torch.int32, device="cuda"),
                              top_p=f(p), min_p=f(mp))
    again, logp2 = R.sample_rows(x, f(u), temperature=f(T), top_k=torch.tensor(k, dtype=torch.int32, device="cuda"),
                                 top_p=f(p), min_p=f(mp))
    assert torch.equal(ids, again) and torch.equal(logp, logp2)
    rows = x.double().cpu().numpy()
    f32 = lambda a: float(np.float32(a))  # noqa: E731
    for r in range(x.shape[0]):
        accepted, want = definition(rows[r], f32(T[r]), k[r], f32(p[r]), f32(mp[r]), f32(u[r]))
        got = int(ids[r])
        assert got in accepted, (r, got, accepted, T[r], k[r], p[r], mp[r], u[r])
        if got == accepted[0]:
            # 64-bit weights to 2^-45 absolute, one f32 rounding of the logarithm
            assert abs(float(logp[r]) - want) <= 2.0 ** -23 * abs(want) + 1e-6, (r, float(logp[r]), want)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 4099, 32001, 151936, 393216])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_match_the_definition(vocab, dtype):
    torch = _cuda()
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 300000 else 6
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * rng.uniform(0.1, 5.0, (rows, 1)).astype(np.float32)
    x = torch.from_numpy(x).cuda().to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype])
    pick = lambda *a: [a[int(i)] for i in rng.integers(0, len(a), rows)]  # noqa: E731
    check(torch, x, pick(1.0, 0.7, 0.05, 2.5, 0.0, 30.0), pick(0, 0, 1, 2, 40, 1000, 5000, vocab, vocab - 1),
          pick(1.0, 1.0, 0.9, 0.5, 0.01, 0.999), pick(0.0, 0.0, 0.0, 0.05, 0.5, 1.0), rng.random(rows).tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [0.5, 1.0, 2.0, 4.0])
@pytest.mark.parametrize("vocab", [1024, 1025, 151936])
def test_borders_among_many_tokens(spread, vocab):
    """Rows without top-k, where thousands of tokens weigh about the same: the border's and the draw's
    neighbourhoods fit one list together, one after the other, or not at all."""
    torch = _cuda()
    rng = np.random.default_rng(int(spread * 10) + vocab)
    rows = 24
    x = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * np.float32(spread)).cuda()
    pick = lambda *a: [a[int(i)] for i in rng.integers(0, len(a), rows)]  # noqa: E731
    check(torch, x, pick(1.0, 0.8, 1.3), [0] * rows, pick(1.0, 0.999, 0.95, 0.9, 0.7), [0.0] * rows,
          rng.random(rows).tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [257, 151936])
def test_ties_infinities_and_nan(vocab):
    torch = _cuda()
    inf, nan = math.inf, math.nan
    x = torch.zeros(16, vocab, device="cuda")            # row 0: all equal
    x[1, ::2] = -0.0                                     # the two zeros are equal
    x[2] = -inf
    x[2, 100] = 1.0                                      # one token left by a mask
    x[3] = -inf                                          # none left
    x[4] = nan
    x[5, 7] = inf
    x[6, 3:] = nan
    x[7] = torch.finfo(torch.float32).min                # a mask of the type's lowest value
    x[8] = torch.finfo(torch.float32).min
    x[8, 5:200:3] = 2.0
    x[9, :] = torch.randint(0, 3, (vocab,), device="cuda").float()      # three large classes of ties
    x[10] = x[9] * 0.01
    x[11] = -torch.arange(vocab, device="cuda").float()                 # weights that run out of range
    x[12] = torch.randn(vocab, device="cuda") * 1e-7                    # values closer than any bin
    x[13] = 1e30 * torch.randn(vocab, device="cuda")
    x[14] = 3e38
    x[14, 9] = -3e38
    x[15, 1::2] = -inf
    for T, k, p, mp in ((1.0, 0, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (0.7, 50, 0.9, 0.0), (1.5, 0, 1.0, 0.1), (1.0, 3, 1.0, 1.0)):
        for u in (0.0, 0.25, 0.5, 0.75, 1.0 - 2.0 ** -24):
            check(torch, x, [T] * 16, [k] * 16, [p] * 16, [mp] * 16, [u] * 16)


@pytest.mark.gpu
def test_settings_outside_their_range_and_left_out():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    x = torch.randn(8, 5000, device="cuda")
    check(torch, x, [-1.0, math.nan, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0], [0, 0, -5, 10 ** 9, 0, 0, 0, 0],
          [1.0, 1.0, 1.0, 1.0, 0.0, -1.0, math.nan, 7.0], [0.0, 0.0, 0.0, 0.0, 0.0, 0.0, math.nan, 2.0], [0.4] * 8)
    u = torch.full((8,), 0.6, device="cuda")
    ids, logp = R.sample_rows(x, u)
    ones = torch.ones(8, device="cuda")
    want = R.sample_rows(x, u, ones, torch.zeros(8, dtype=torch.int32, device="cuda"), ones, 0 * ones)
    assert torch.equal(ids, want[0]) and torch.equal(logp, want[1])


@pytest.mark.gpu
def test_strided_rows_other_stream_and_replay():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    wide = torch.randn(5, 7003, device="cuda")
    x = wide[:, 1:7002]                       # rows that start at any alignment
    u = torch.rand(5, device="cuda")
    p = torch.full((5,), 0.8, device="cuda")
    want = R.sample_rows(x.contiguous(), u, top_p=p)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = R.sample_rows(x, u, top_p=p, stream=s)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ids = torch.zeros(5, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, logp = R.sample_rows(x, u, top_p=p, ids=ids)
    for seed in range(2):
        wide.copy_(torch.randn(5, 7003, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = R.sample_rows(x.contiguous(), u, top_p=p)
        assert torch.equal(ids, want[0]) and torch.equal(logp, want[1])
    assert R.sample_rows(x[:0], u[:0])[0].numel() == 0


@pytest.mark.gpu
def test_draws_follow_the_softmax():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    n = 4096
    x = torch.tensor([1.0, 0.2, -0.5, 2.0, 0.0], device="cuda").repeat(n, 1)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    ids, _ = R.sample_rows(x, u.float(), temperature=torch.full((n,), 0.8, device="cuda"))
    share = torch.bincount(ids.long(), minlength=5).double() / n
    assert float((share - torch.softmax(x[0].double() / 0.8, 0)).abs().max()) <= 1.0 / n   # one stratum a border


@pytest.mark.gpu
@pytest.mark.parametrize("u", [0.5, 0.99995, 1.0 - 2.0 ** -24])
@pytest.mark.parametrize("tail", ["uniform", "deep"])
def test_borders_at_the_end_of_heavy_rows(tail, u):
    """Rows whose weights add up to thousands of times the largest one, with the border or the draw among
    the last of them: the sum, about 2^56 units, is no exact double, and rounds up in every other row."""
    torch = _cuda()
    rng = np.random.default_rng(3)
    rows, vocab = 16, 151936
    if tail == "uniform":
        x = rng.uniform(-25.0, 0.0, (rows, vocab))
    else:
        x = rng.standard_normal((rows, vocab))
        x[:, rng.permutation(vocab)[:1000]] -= 20.0
    x = torch.from_numpy(x.astype(np.float32)).cuda()
    p = [[1.0, 0.9999, 0.99999, 1.0 - 2.0 ** -24][r % 4] for r in range(rows)]
    check(torch, x, [1.0] * rows, [0] * rows, p, [0.0] * rows, [u] * rows)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [3e-33, 1e-36, 1e-40])
@pytest.mark.parametrize("vocab", [700, 5000, 151936])
def test_rows_and_temperatures_near_the_smallest_numbers(vocab, scale):
    """Differences and temperatures below 1e-33, subnormal ones among them: the weights are ordinary."""
    torch = _cuda()
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 100000 else 8
    x = rng.standard_normal((rows, vocab)) * 3.0
    x -= np.where(rng.random(x.shape) < 0.5, rng.uniform(40.0, 4000.0, x.shape), 0.0)  # half of them weigh nothing
    x = torch.from_numpy((x * scale).astype(np.float32)).cuda()
    pick = lambda *a: [a[int(i)] for i in rng.integers(0, len(a), rows)]  # noqa: E731
    check(torch, x, [(1.0, 0.3)[r % 2] * scale for r in range(rows)], pick(0, 0, 0, 40, 2000), pick(1.0, 0.9, 0.5),
          pick(0.0, 0.0, 0.05), rng.random(rows).tolist())
