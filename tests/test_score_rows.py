"""qd_score_rows: log probability of a given token, entropy and the largest tokens per row of logits, against the
definition in 64 bits.

Tolerances (d = mean of max - x under the softmax): a term e^(x - max) is off by 2^-22 (exponential) and by the
rounding of its argument, 2^-22 of it in all; a thread adds count = vocab / (512 C) of them (half a step each) and its
sums are brought to another maximum up to 17 times (5 joins in a warp, 4 in a CTA, 7 in a cluster, and the loop's), an
exponential each: rel = 2^-22 (d + 1 + 17) + count 2^-24 of the sum S. Logarithms are off by rel + 2^-23 of what is
added up; the entropy's quotient by 2 rel d more. (A thread's running maximum moves a few times on the way: 8 more.)"""
import math

import numpy as np
import pytest

from kernel_optimization_webgpu_b200 import _lib


def test_arguments_are_refused():
    L = _lib.load()
    p = 4096
    ok = dict(logits=p, dtype=1, rows=1, vocab=10, stride=10, tokens=p, top=2, logp=p, ent=p, ids=p, tops=p)

    def call(**kw):
        c = {**ok, **kw}
        return L.qd_score_rows(c["logits"], c["dtype"], c["rows"], c["vocab"], c["stride"], c["tokens"], c["top"], c["logp"],
                               c["ent"], c["ids"], c["tops"], None)

    for bad in (dict(rows=-1), dict(vocab=0), dict(dtype=5), dict(dtype=-1), dict(stride=9), dict(top=-1), dict(top=65, vocab=100, stride=100),
                dict(top=11), dict(logits=None), dict(tokens=None), dict(logp=None), dict(ids=None), dict(tops=None)):
        assert call(**bad) == _lib.QD_E_INVALID, bad
    assert call(vocab=(1 << 30) + 1, stride=1 << 31) == _lib.QD_E_RANGE
    assert call(rows=0, logits=None, tokens=None, logp=None) == _lib.QD_OK


def test_outputs_over_their_inputs_are_refused():
    """Two rows of ten f32 logits, 48 bytes apart, at 1 << 40; tokens at 1 << 41. (What is not refused is ended by vocab.)"""
    L = _lib.load()
    at, far = 1 << 40, 1 << 42
    ok = dict(logits=at, tokens=1 << 41, logp=far, ent=far + 64, ids=far + 128, tops=far + 192)

    def call(vocab=10, **kw):
        c = {**ok, **kw}
        rc = L.qd_score_rows(c["logits"], 1, 2, vocab, 12, c["tokens"], 2, c["logp"], c["ent"], c["ids"], c["tops"], None)
        return rc, L.qd_last_error(None)

    for bad in (dict(logp=at), dict(ent=at + 84), dict(ids=at - 12), dict(tops=at + 60), dict(logp=1 << 41), dict(ids=(1 << 41) - 8)):
        rc, said = call(**bad)
        assert rc == _lib.QD_E_INVALID and b"overlaps" in said, bad


def test_python_wrapper_refuses():
    torch = pytest.importorskip("torch")
    from kernel_optimization_webgpu_b200 import runtime as R
    x, t = torch.zeros(2, 9), torch.zeros(2, dtype=torch.int32)
    for args, kw in (((x[0], t), {}), ((x, t[:1]), {}), ((x, t.long()), {}), ((x.t(), t), {}), ((x.long(), t), {}),
                     ((x, t), dict(top=65)), ((x, t), dict(top=-1)), ((x, t), {})):
        with pytest.raises(ValueError):
            R.score_rows(*args, **kw)


def _cuda():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def check(torch, x, tokens, top):
    from kernel_optimization_webgpu_b200 import runtime as R
    rows, V = x.shape
    t = torch.tensor(tokens, dtype=torch.int32, device="cuda")
    logp, ent, ids, tops = R.score_rows(x, t, top=top)
    again = R.score_rows(x, t, top=top)
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip((logp, ent, ids, tops), again))
    v = x.double().cpu().numpy()
    logp, ent, ids, tops = (a.cpu().numpy() for a in (logp, ent, ids, tops))
    for r in range(rows):
        key = np.where(np.isnan(v[r]), -np.inf, v[r])
        order = np.lexsort((np.arange(V), np.isnan(v[r]), -key))[:top]
        assert ids[r].tolist() == order.tolist(), (r, ids[r], order)
        if not np.isfinite(key.max()) or np.isnan(v[r]).any():
            assert np.isnan(logp[r]) and np.isnan(ent[r]) and np.isnan(tops[r]).all(), r
            continue
        d = key - key.max()
        e = np.exp(d)
        S = e.sum()
        far = np.where(e > 0, d, 0.0)
        mean = float(-(far * e).sum() / S)
        want = d - math.log(S)
        h = math.log(S) + mean
        rel = 2.0 ** -22 * (mean + 26) + (V / 512 / max(1, min(8, V // 2048)) + 8) * 2.0 ** -24
        assert abs(ent[r] - h) <= rel * (1 + 2 * mean) + 2.0 ** -22 * (abs(math.log(S)) + mean), (r, ent[r], h)
        for got, w in [(logp[r], want[tokens[r]] if 0 <= tokens[r] < V else math.nan)] + list(zip(tops[r], want[order])):
            if math.isnan(w) or math.isinf(w):
                assert math.isnan(got) if math.isnan(w) else got == w, (r, got, w)
            else:
                assert abs(got - w) <= rel + 2.0 ** -23 * (abs(w) + abs(math.log(S))), (r, got, w)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 33, 127, 1000, 4099, 32001, 151936, 393216])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("top", [0, 1, 20, 64])
def test_rows_match_the_definition(vocab, dtype, top):
    torch = _cuda()
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 100000 else 5
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * rng.uniform(0.1, 5.0, (rows, 1)).astype(np.float32)
    x = torch.from_numpy(x).cuda().to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype])
    tokens = rng.integers(0, vocab, rows).tolist()
    tokens[:4] = [0, vocab - 1, int(x[2].argmax()), int(x[3].argmin())]
    check(torch, x, tokens, min(top, vocab))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 40, 300, 1000])
def test_any_number_of_rows(rows):
    torch = _cuda()
    x = torch.randn(rows, 5003, device="cuda") * 2
    check(torch, x, [(r * 37) % 5003 for r in range(rows)], 5)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [257, 20011, 151936])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_ties_masks_infinities_and_nan(vocab, top):
    torch = _cuda()
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.zeros(20, vocab, device="cuda")            # row 0: all equal
    x[1, ::2] = -0.0                                     # the two zeros are equal
    x[2] = -inf
    x[2, 100] = 1.0                                      # one token left by a mask
    x[3] = -inf                                          # none left
    x[4] = nan
    x[5, 7] = inf
    x[6, 3:] = nan
    x[7] = low                                           # a mask of the type's lowest value
    x[8] = low
    x[8, 5:200:3] = 2.0
    x[9] = torch.randint(0, 3, (vocab,), generator=g, device="cuda").float()   # three large classes of ties
    x[10] = x[9] * 0.01
    x[11] = -torch.arange(vocab, device="cuda").float()  # weights that run out of range
    x[12] = torch.arange(vocab, device="cuda").float() * 0.01                  # ascending: the largest come last
    x[13] = 1e30 * torch.randn(vocab, generator=g, device="cuda")
    x[14] = 3e38
    x[14, 9] = -3e38
    x[15, 1::2] = -inf
    x[16] = torch.randn(vocab, generator=g, device="cuda")
    x[16, vocab // 2:] = -inf                            # a slice with nothing in it
    x[17] = -inf
    x[17, 30:250:7] = torch.randn(32, generator=g, device="cuda")              # a few in one place
    x[18] = x[16]
    x[18, vocab - 1] = nan
    x[19] = torch.randn(vocab, generator=g, device="cuda").round()
    x[19, 40:104] = 50.0                                 # 64 equal ones side by side
    check(torch, x, [100] * 18 + [-1, vocab], top)
    check(torch, x.bfloat16(), [5] * 20, top)


@pytest.mark.gpu
def test_all_of_a_small_vocabulary():
    torch = _cuda()
    x = torch.randn(6, 64, device="cuda")
    x[1, 5:] = -math.inf
    x[2, 9:] = math.nan
    x[3] = 0.0
    x[4, ::3] = -math.inf
    x[5, ::3] = math.nan
    check(torch, x, [0, 1, 2, 3, 4, -7], 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_rows_at_any_alignment_other_stream_and_replay(dtype):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    T = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    for first in range(1, 9):
        wide = torch.full((5, 7011), 99.0, device="cuda").to(T)      # what lies beside a row is larger than all of it
        wide[:, first:first + 7000] = torch.randn(5, 7000, device="cuda").to(T)
        check(torch, wide[:, first:first + 7000], [0, 6999, 3, 4, 5], 10)
    x = wide[:, 8:7008]
    t = torch.arange(5, dtype=torch.int32, device="cuda")
    want = R.score_rows(x.contiguous(), t, top=7)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = R.score_rows(x, t, top=7, stream=s)
    s.synchronize()
    assert torch.equal(got[2], want[2])
    logp = torch.zeros(5, device="cuda")
    ids = torch.zeros(5, 7, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        R.score_rows(x, t, top=7, logprobs=logp, top_ids=ids)
    for _ in range(2):
        wide.copy_(torch.randn(5, 7011, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = R.score_rows(x, t, top=7)
        assert torch.equal(logp, want[0]) and torch.equal(ids, want[2])
    assert R.score_rows(x[:0], t[:0], top=3)[2].shape == (0, 3)
    with pytest.raises(ValueError):
        R.score_rows(x, t, top=7, top_ids=ids[:, :6])


@pytest.mark.gpu
def test_scores_of_draws_are_the_samplers():
    """With neither cut nor temperature the sampler's logarithm is this one."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    x = torch.randn(64, 151936, device="cuda") * 3
    ids, logp = R.sample_rows(x, torch.rand(64, device="cuda"))
    assert float((R.score_rows(x, ids)[0] - logp).abs().max()) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("offset,size", [(1000.0, 4.0), (-30000.0, 1.0), (3.0e6, 100.0), (0.0, 1e-30)])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_rows_with_a_common_offset(offset, size, top):
    """A softmax does not change under an offset, and the time does not either: distinct values next to each other are
    told apart by their last bits, not one pass after the other (which took more than ten times as long)."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    g = torch.Generator(device="cuda").manual_seed(3)
    plain = torch.randn(6, 151936, generator=g, device="cuda")
    x = plain * size + offset
    tokens = [5, 151935, 0, int(x[3].argmax()), 77, 1000]
    check(torch, x, tokens, top)
    t = torch.tensor(tokens, dtype=torch.int32, device="cuda")

    def us(rows):
        best = math.inf
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(20):
                R.score_rows(rows, t, top=top)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert us(x) < 2 * us(plain)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [19, 20, 21, 40])
def test_many_tokens_above_nothing(top):
    """Positive tokens in 20 of the 128 groups of a row's threads, and 40 of the 256 threads, only (columns 0..159 of
    every 1024), all others negative: they are not looked through one after the other, which took 30 to 60 times the time
    of other rows. Twice covers the second look at them, as much again the ordering of up to 1024 that are listed."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    g = torch.Generator(device="cuda").manual_seed(8)
    rows = 600   # one block a row
    plain = torch.randn(rows, 32000, generator=g, device="cuda")
    x = plain.abs() + 0.1
    x[:, torch.arange(32000, device="cuda") % 1024 >= 160] *= -1
    t = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ids = R.score_rows(x, t, top=top)[2]
    want = x.topk(top, -1)
    assert torch.equal(x.gather(1, ids.long()), want.values)
    check(torch, x[:3], [0, 1, 2], top)

    def us(rows):
        best = math.inf
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                R.score_rows(rows, t, top=top)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert us(x) < 4 * us(plain)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows 4.4 GB apart."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    wide = 2 ** 30 + 2 ** 26
    x = torch.empty(wide + 5000, device="cuda").as_strided((2, 5000), (wide, 1))
    x.copy_(torch.randn(2, 5000, device="cuda"))
    t = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    for a, b in zip(R.score_rows(x, t, top=4), R.score_rows(x.contiguous(), t, top=4)):
        assert torch.allclose(a, b, atol=1e-5) if a.is_floating_point() else torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,allowed", [(151936, 5000), (151936, 1500), (151936, 1030), (40000, 3000)])
@pytest.mark.parametrize("top", [5, 20, 64])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masks_that_leave_neighbours(vocab, allowed, top, dtype):
    """A mask that leaves a range of token ids, which few of a row's groups of threads hold."""
    torch = _cuda()
    g = torch.Generator(device="cuda").manual_seed(allowed)
    x = torch.full((6, vocab), -math.inf, device="cuda")
    for r, first in enumerate((0, 7, 20001, vocab - allowed, 19000, 100)):
        x[r, first:first + allowed] = torch.randn(allowed, generator=g, device="cuda") * 3
    x[5, 100:100 + allowed:2] = 2.0   # half of them alike
    check(torch, x.to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype]), [1, 8, 20002, vocab - 1, 19000, 100], top)
