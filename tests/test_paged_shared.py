"""Decode attention over shared prefixes (qd_paged_attn_decode_shared): refusals on the host (no GPU), and the CUDA
path against the plain 64-bit evaluation of test_paged.py, whose tolerances it takes (the shared positions' products are
the prompt's, the others' the decoding step's; their join adds three roundings of an exponential, 2^-20)."""
import math

import pytest

from kernel_optimization_webgpu_b200 import _lib
from test_paged import BAD_CACHES, BASE, D, HALF_STEP, HEADS, _cuda, _kv, _types, close, make_cache, plain_attention


def test_arguments_are_refused():
    L = _lib.load()
    ok = dict(kv=_kv(), q=BASE, dtype=1, stride=256, heads=2, groups=1, starts=4096, shared=4096, scale=0.0, y=2 * BASE,
              y_stride=256, ws=4096)

    def call(**kw):
        c = {**ok, **kw}
        return L.qd_paged_attn_decode_shared(c["kv"], c["q"], c["dtype"], c["stride"], c["heads"], c["groups"], c["starts"],
                                             c["shared"], c["scale"], c["y"], c["y_stride"], c["ws"], None)

    for bad in [dict(q=None), dict(y=None), dict(ws=None), dict(ws=4104), dict(q=BASE + 8), dict(dtype=2), dict(dtype=9),
                dict(stride=248), dict(y_stride=128), dict(heads=3), dict(heads=130, stride=130 * 128, y_stride=130 * 128),
                dict(scale=math.inf), dict(groups=-1), dict(groups=3), dict(starts=None), dict(shared=None), dict(y=BASE),
                dict(y=4096), dict(kv=None)] + [dict(kv=_kv(**b)) for b in BAD_CACHES]:
        assert call(**bad) == _lib.QD_E_INVALID, bad
    assert call(groups=0) == _lib.QD_OK and call(kv=_kv(batch=0), groups=0) == _lib.QD_OK   # nothing to do
    assert call(kv=_kv(batch=4096, table_width=1 << 22, table_stride=1 << 22, block_table=64, seq_lens=64)) == _lib.QD_E_RANGE
    size = L.qd_paged_attn_decode_shared_workspace_bytes
    assert size(64, 1, 16, 8) > 0 and size(2, 3, 16, 8) == 0 and size(-1, 0, 16, 8) == 0 and size(2, 1, 16, 5) == 0


def test_python_wrapper_refuses_before_it_enqueues():
    torch = pytest.importorskip("torch")
    from kernel_optimization_webgpu_b200 import runtime as R
    k = torch.zeros(4, 2, 16, D, dtype=torch.float16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    q, starts = torch.zeros(2, 2, D), torch.tensor([0, 2], dtype=torch.int32)
    for args in ((q, k, k, table, lens, starts, lens), (q, k, k, table, lens, starts.long(), lens),
                 (q, k, k, table, lens, starts, lens[:1]), (q[:1], k, k, table, lens, starts, lens)):
        with pytest.raises(ValueError):
            R.paged_attn_decode_shared(*args)


def make_shared(torch, sizes, prefix, tails, page, kv_heads, cache, seed=0):
    """Groups of sizes[i] sequences sharing prefix[i] positions, with tails[b] of their own; pages of a prefix are
    listed by its group's first sequence only (the others' entries there are out of the pool), but for the page in which
    it ends. (k, v, table, lens, starts, shared, whole): whole: the table with everything filled in."""
    held = [p for p, m in zip(prefix, sizes) for _ in range(m)]
    lead = [sum(sizes[:i]) for i, m in enumerate(sizes) for _ in range(m)]
    lens = [h + t for h, t in zip(held, tails)]
    k, v, table, n = make_cache(torch, lens, page, kv_heads, cache, seed=seed, fill=math.nan)
    whole = table.clone()
    for b in range(len(lens)):
        if lead[b] == b:
            continue
        full, rest = held[b] // page, held[b] % page
        whole[b, :full] = table[lead[b], :full]
        table[b, :full] = -7 if b % 2 else 10 ** 6
        if rest:   # its own copy of the page in which the prefix ends
            for x in (k, v):
                x[table[b, full], :, :rest] = x[table[lead[b], full], :, :rest]
    cum = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    dev = dict(dtype=torch.int32, device="cuda")
    return k, v, table, n, torch.tensor(cum, **dev), torch.tensor(held, **dev), whole


CASES = [([4], [1000], [40] * 4), ([1], [300], [20]), ([2, 1, 3], [70, 500, 0], [1, 30, 2, 1, 200, 64]),
         ([9, 5], [128, 1300], [1] * 14), ([3], [15], [5, 0, 1]), ([300], [257], [1 + i % 9 for i in range(300)]),
         ([2] * 40, [100 + 3 * i for i in range(40)], [1 + i % 50 for i in range(80)]), ([4], [4000], [700, 1, 64, 0]),
         ([5], [0], [10, 1, 700, 64, 65])]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}groups{sum(c[0])}of{max(c[1])}")
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: f"{h[0]}q{h[1]}kv")
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
def test_shared(case, heads, io, cache):
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    sizes, prefix, tails = case
    page = [16, 32, 64, 256][(len(tails) + heads[0]) % 4]
    k, v, table, n, starts, shared, whole = make_shared(torch, sizes, prefix, tails, page, heads[1], cache, seed=len(tails))
    q = (torch.randn(len(tails), heads[0], D, device="cuda") * 1.5).to(_types(torch)[io])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = R.paged_attn_decode_shared(q, k, v, table, n, starts, shared, status=status)
    assert int(status) == 0
    want, tol = plain_attention(torch, q, k, v, whole, n, [1] * len(tails), 0, 0, D ** -0.5, io, cache)
    close(torch, y, want, tol + 2.0 ** -20 * want.abs().amax(-1, keepdim=True))
    assert torch.equal(R.paged_attn_decode_shared(q, k, v, table, n, starts, shared), y)


@pytest.mark.gpu
@pytest.mark.parametrize("io", ["f32", "f16"])
def test_shared_lengths_of_any_size(io):
    """Lengths below, at and beyond the shared ones, negative and unequal ones within a group: position j of
    sequence b is looked up in the first sequence's row when j < shared_lens[b]."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    lens = [300, 20, 0, 250, 129, 128, 127, 1, 300, 300]
    k, v, table, n = make_cache(torch, [300] * 10, 16, 2, "f16")
    n.copy_(torch.tensor(lens, dtype=torch.int32))
    shared = torch.tensor([200, 200, 200, 10 ** 9, 128, 129, -5, 0, 2 ** 31 - 1, 33], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 4, 4, 8, 9, 10], dtype=torch.int32, device="cuda")
    lead = [0, 0, 0, 0, 4, 4, 4, 4, 8, 9]
    q = torch.randn(10, 4, D, device="cuda").to(_types(torch)[io])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = R.paged_attn_decode_shared(q, k, v, table, n, starts, shared, status=status)
    assert int(status) == 0 and bool((y[2] == 0).all())
    # a cache in which every sequence holds its rows by itself
    kk, vv = (x[table.long()].transpose(2, 3).reshape(10, -1, 2, D) for x in (k, v))
    j = torch.arange(kk.shape[1], device="cuda")
    mine = j[None] >= shared[:, None]
    kk, vv = (torch.where(mine[..., None, None], x, x[lead]).reshape(10, -1, 16, 2, D).transpose(2, 3).flatten(0, 1).contiguous()
              for x in (kk, vv))
    own = torch.arange(kk.shape[0], dtype=torch.int32, device="cuda").view(10, -1)
    want, tol = plain_attention(torch, q, kk, vv, own, n, [1] * 10, 0, 0, D ** -0.5, io, "f16")
    close(torch, y, want, tol + 2.0 ** -20 * want.abs().amax(-1, keepdim=True))


@pytest.mark.gpu
def test_padding_sequences_strides_scale_and_stream():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n, starts, shared, whole = make_shared(torch, [3, 2], [300, 40], [20, 1, 99, 7, 64], 32, 2, "f16")
    pad = 3   # sequences behind the last group: garbage that nobody looks at
    table = torch.cat([table, torch.full((pad, table.shape[1]), 10 ** 9, dtype=torch.int32, device="cuda")])
    n2 = torch.cat([n, torch.tensor([2 ** 31 - 1, -4, 5], dtype=torch.int32, device="cuda")])
    shared = torch.cat([shared, torch.tensor([7, 2 ** 31 - 1, -1], dtype=torch.int32, device="cuda")])
    wide = torch.randn(8, 8 * D + 64, device="cuda")
    wide[5:] = math.nan
    q = wide[:, :8 * D].unflatten(1, (8, D))
    out = torch.full((8, 8 * D + 8), 7.0, device="cuda")
    y = out[:, :8 * D].unflatten(1, (8, D))
    size = _lib.load().qd_paged_attn_decode_shared_workspace_bytes(8, 2, 8, 2)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    R.paged_attn_decode_shared(q, k, v, table, n2, starts, shared, scale=-0.3, y=y, workspace=ws, status=status, stream=s)
    s.synchronize()
    assert int(status) == 0 and bool((out[5:] == 7.0).all()) and bool((out[:, 8 * D:] == 7.0).all())
    want, tol = plain_attention(torch, q[:5], k, v, whole, n, [1] * 5, 0, 0, -0.3, "f32", "f16")
    close(torch, y[:5], want, tol + 2.0 ** -20 * want.abs().amax(-1, keepdim=True))
    with pytest.raises(ValueError, match="workspace"):
        R.paged_attn_decode_shared(q, k, v, table, n2, starts, shared, workspace=ws[:-1])
    with pytest.raises(ValueError, match="overlaps"):
        R.paged_attn_decode_shared(q, k, v, table, n2, starts, shared, y=q)
    # no group: nothing is done
    y.fill_(7.0)
    R.paged_attn_decode_shared(q, k, v, table, n2, starts[:1], shared, y=y)
    assert bool((y == 7.0).all())


@pytest.mark.gpu
def test_bad_pages_and_lengths_are_left_out_and_flagged():
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n, starts, shared, whole = make_shared(torch, [3], [160], [30, 20, 1], 16, 2, "f16")
    q = torch.randn(3, 4, D, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run():
        status.zero_()
        return R.paged_attn_decode_shared(q, k, v, table, n, starts, shared, status=status)

    def plain(drop):
        ys = []
        for b in range(3):
            j = torch.arange(int(n[b]), device="cuda")
            j = j[~torch.isin(j // 16, torch.tensor(drop[b], device="cuda"))]
            pg = whole[b].long()[j // 16]
            kk, vv = (x[pg, :, j % 16].double().repeat_interleave(2, 1) for x in (k, v))
            ys.append(torch.einsum("hj,jhd->hd", torch.softmax(torch.einsum("hd,jhd->hj", q[b].double(), kk) / math.sqrt(D), -1), vv))
        return torch.stack(ys)

    good = table.clone()
    table[0, 4] = -1          # of the prefix: left out for all
    y = run()
    assert int(status) == _lib.QD_PAGED_BAD_PAGE and float((y.double() - plain([[4], [4], [4]])).abs().max()) < 1e-4
    table.copy_(good)
    table[1, 11] = 10 ** 6    # of a sequence's own
    y = run()
    assert int(status) == _lib.QD_PAGED_BAD_PAGE and float((y.double() - plain([[], [11], []])).abs().max()) < 1e-4
    table.copy_(good)
    keep = n.clone()
    n[1] = 10 ** 9            # cut to the table, whose unused entries are none
    y = run()
    assert int(status) & _lib.QD_PAGED_BAD_LENGTH
    n.copy_(keep)
    assert float((y[0].double() - plain([[], [], []])[0]).abs().max()) < 1e-4
    n[1] = -1
    assert bool((run()[1] == 0).all()) and int(status) == _lib.QD_PAGED_BAD_LENGTH


@pytest.mark.gpu
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("groups", [2, 60])
def test_a_block_that_gives_up_leaves_nan_and_a_status(io, cache, groups):
    """Block 0 (the last rows of the last group, the first KV head) withholds its first key tile. 60 groups: blocks take
    the work of others."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n, starts, shared, _ = make_shared(torch, [3] * groups, [900] * groups, [9] * (3 * groups), 64, 4, cache)
    q = torch.randn(3 * groups, 8, D, device="cuda").to(_types(torch)[io])
    want = R.paged_attn_decode_shared(q, k, v, table, n, starts, shared)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.load().qd_paged_inject_stall()
    y = R.paged_attn_decode_shared(q, k, v, table, n, starts, shared, status=status)
    gone = y.isnan().any(-1)
    assert int(status) == _lib.QD_PAGED_TIMEOUT and torch.equal(gone, y.isnan().all(-1))
    assert bool(gone[-3:, :2].all()) and int(gone.sum()) == 6
    assert torch.equal(y[~gone], want[~gone])
    status.zero_()
    assert torch.equal(R.paged_attn_decode_shared(q, k, v, table, n, starts, shared, status=status), want) and int(status) == 0


@pytest.mark.gpu
def test_replays_follow_lengths_and_groups():
    """Two graphs with workspaces of their own; the groups and lengths change between replays."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n = make_cache(torch, [700] * 6, 16, 2, "f16")
    table[1:] = torch.where(torch.arange(table.shape[1], device="cuda") < 30, table[0], table[1:])   # all share 480 positions
    starts = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    shared = torch.full((6,), 480, dtype=torch.int32, device="cuda")
    q = torch.randn(6, 8, D, device="cuda")
    size = _lib.load().qd_paged_attn_decode_shared_workspace_bytes(6, 2, 8, 2)
    ys, graphs, spaces = [], [], []
    for i in range(2):
        spaces.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
        ys.append(torch.zeros_like(q))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            R.paged_attn_decode_shared(q, k, v, table, n, starts, shared, y=ys[i], workspace=spaces[i])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for lens, cut, held in (([700] * 6, 3, 480), ([500, 480, 3, 0, 481, 699], 1, 480), ([700, 20, 650, 481, 512, 640], 6, 100)):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        starts[1] = cut
        shared.fill_(held)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        want, tol = plain_attention(torch, q, k, v, table, n, [1] * 6, 0, 0, D ** -0.5, "f32", "f16")
        for y in ys:
            close(torch, y, want, tol + 2.0 ** -20 * want.abs().amax(-1, keepdim=True))


@pytest.mark.gpu
def test_answers_to_one_prompt_step_by_step():
    """A prompt appended once, its pages shared by five sequences that grow token by token, scored and drawn."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    torch.manual_seed(2)
    H, kvh, page, B, prompt = 8, 2, 16, 5, 75
    k, v = (torch.full((40, kvh, page, D), math.nan, device="cuda", dtype=torch.float16) for _ in "kv")
    order = torch.randperm(40, device="cuda").to(torch.int32)
    table = torch.full((B, 8), -1, dtype=torch.int32, device="cuda")
    table[0, :5] = order[:5]
    one = torch.tensor([prompt], dtype=torch.int32, device="cuda")
    starts1 = torch.tensor([0, prompt], dtype=torch.int32, device="cuda")
    q = R.paged_append(torch.randn(prompt, (H + 2 * kvh) * D, device="cuda"), k, v, table[:1], one, None, None, H, q_starts=starts1)
    R.paged_attn_prompt(q.view(-1, H, D), k, v, table[:1], one, starts1)
    for b in range(1, B):   # the prefix's full pages are shared, the page in which it ends is copied
        table[b, 4] = order[5 + b]
        k[table[b, 4]], v[table[b, 4]] = k[table[0, 4]], v[table[0, 4]]
    table[:, 5:7] = order[20:30].view(B, 2)
    lens = torch.full((B,), prompt, dtype=torch.int32, device="cuda")
    shared, starts = lens.clone(), torch.tensor([0, B], dtype=torch.int32, device="cuda")
    whole = table.clone()
    whole[:, :4] = table[0, :4]
    head = torch.randn(H * D, 1003, device="cuda") * 0.05
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for step in range(20):
        lens += 1
        q = R.paged_append(torch.randn(B, (H + 2 * kvh) * D, device="cuda"), k, v, table, lens, None, None, H, status=status)
        y = R.paged_attn_decode_shared(q.view(B, H, D), k, v, table, lens, starts, shared, status=status)
        want, tol = plain_attention(torch, q.view(B, H, D), k, v, whole, lens, [1] * B, 0, 0, D ** -0.5, "f32", "f16")
        close(torch, y, want, tol + 2.0 ** -20 * want.abs().amax(-1, keepdim=True))
        logits = y.reshape(B, -1) @ head
        ids, _ = R.sample_rows(logits, torch.rand(B, device="cuda"))
        logp, _, top, _ = R.score_rows(logits, ids, top=3)
        exact = torch.log_softmax(logits.double(), -1)
        assert float((logp - exact.gather(1, ids.long()[:, None])[:, 0]).abs().max()) < 1e-5
        assert torch.equal(top[:, 0].long(), logits.argmax(-1))
    assert int(status) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,prefix", [([3], [200]), ([40], [600]), ([2] * 40, [130 + 3 * i for i in range(40)])],
                         ids=["one", "wide", "many"])
@pytest.mark.parametrize("io", ["f16", "bf16"])
def test_16_bit_queries_keep_both_parts_of_a_weight(sizes, prefix, io):
    """Values of alternating sign under nearly equal weights: what rounding a weight to 16 bits (2^-11, 2^-8) would
    leave does not cancel, the output and its own rounding do. The tolerance is that of two parts (f32 queries' terms),
    and the output's half step."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n, starts, shared, whole = make_shared(torch, sizes, prefix, [1 + b % 5 for b in range(sum(sizes))], 16, 2, io)
    v[:, :, ::2] = v[:, :, ::2].abs()
    v[:, :, 1::2] = -v[:, :, 1::2].abs()
    q = (torch.randn(sum(sizes), 8, D, device="cuda") * 0.02).to(_types(torch)[io])
    y = R.paged_attn_decode_shared(q, k, v, table, n, starts, shared)
    want, tol = plain_attention(torch, q, k, v, whole, n, [1] * sum(sizes), 0, 0, D ** -0.5, "f32", io)
    tol = tol + HALF_STEP[io] * want.abs() + (2.0 ** -25 if io == "f16" else 0.0) + 2.0 ** -20 * want.abs().amax(-1, keepdim=True)
    close(torch, R.paged_attn_decode(q, k, v, whole, n), want, tol)
    close(torch, y, want, tol)


def test_places_to_stall_at_are_checked():
    L = _lib.load()
    for bad in (0, -1, 99):
        assert L.qd_paged_inject_stall_at(bad) == _lib.QD_E_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("prefix", [200, 400, [100 + 40 * (i % 9) for i in range(120)]], ids=["two", "four", "ragged"])
def test_threads_that_begin_late_change_nothing(io, cache, prefix):
    """One set of a block's threads may be a whole row tile ahead of the other: here it has 40 us at every tile, more
    than a tile of 2 to 4 key tiles takes. 120 groups of 4 KV heads: blocks take others' work."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    groups = 120
    prefix = [prefix] * groups if isinstance(prefix, int) else prefix
    k, v, table, n, starts, shared, _ = make_shared(torch, [2] * groups, prefix, [3] * (2 * groups), 64, 4, cache)
    q = torch.randn(2 * groups, 8, D, device="cuda").to(_types(torch)[io])
    want = R.paged_attn_decode_shared(q, k, v, table, n, starts, shared)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert _lib.load().qd_paged_inject_stall_at(_lib.QD_PAGED_STALL_LATE) == _lib.QD_OK
    y = R.paged_attn_decode_shared(q, k, v, table, n, starts, shared, status=status)
    assert int(status) == 0 and torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("prefix", [100, 900])
@pytest.mark.parametrize("groups", [200, 700])
def test_rows_that_a_block_took_and_could_not_begin_are_nan(io, cache, prefix, groups):
    """Groups of one KV head: block 0 has the last group's rows and takes another group's before it gives up (of 700
    for certain: 148 blocks run and ask once each while 552 are left; of 200, 52 are left for all who ask, and it may
    come too late). The workspace holds zeros, as a place among the sums zero of them."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    k, v, table, n, starts, shared, _ = make_shared(torch, [3] * groups, [prefix] * groups, [9] * (3 * groups), 64, 1, cache)
    q = torch.randn(3 * groups, 4, D, device="cuda").to(_types(torch)[io])
    want = R.paged_attn_decode_shared(q, k, v, table, n, starts, shared)
    ws = torch.zeros(_lib.load().qd_paged_attn_decode_shared_workspace_bytes(3 * groups, groups, 4, 1), dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert _lib.load().qd_paged_inject_stall_at(_lib.QD_PAGED_STALL_LAST) == _lib.QD_OK
    y = R.paged_attn_decode_shared(q, k, v, table, n, starts, shared, workspace=ws, status=status)
    assert int(status) == _lib.QD_PAGED_TIMEOUT
    gone = y.isnan().all(-1).view(groups, 12)
    assert torch.equal(gone, y.isnan().any(-1).view(groups, 12))
    assert bool(gone[-1].all()) and torch.equal(gone.any(-1), gone.all(-1))
    assert int(gone.any(-1).sum()) in ((1, 2) if groups == 200 else (2,))
    keep = ~gone.view(-1, 4)
    assert torch.equal(y[keep], want[keep])
    status.zero_()
    assert torch.equal(R.paged_attn_decode_shared(q, k, v, table, n, starts, shared, workspace=ws, status=status), want)
    assert int(status) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_what_was_written_right_before_is_seen(captured):
    """Steps of append and attention without a pause, each step's new rows, lengths and queries written by the launches
    just before: the results of the same calls made one at a time. One workspace for all, with old contents."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    H, kvh, B, steps = 8, 2, 24, 40
    k, v, table, n, starts, shared, whole = make_shared(torch, [10, 14], [300, 77], [1] * B, 16, kvh, "f16")
    grown = torch.arange(k.shape[0], k.shape[0] + 4 * B, dtype=torch.int32, device="cuda").view(B, 4)   # pages to grow into
    k, v = (torch.cat([x, torch.zeros(4 * B, kvh, 16, D, dtype=x.dtype, device="cuda")]) for x in (k, v))
    table = torch.cat([table, torch.full((B, 4), -1, dtype=torch.int32, device="cuda")], 1)
    for b in range(B):
        used = -(-int(n[b]) // 16)
        table[b, used:used + 4] = grown[b]
    qkv = torch.randn(steps, B, (H + 2 * kvh) * D, device="cuda")
    ws = torch.full((_lib.load().qd_paged_attn_decode_shared_workspace_bytes(B, 2, H, kvh),), 255, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    keep = [x.clone() for x in (k, v, n)]

    def run(pause):
        ys = []
        for i in range(steps):
            n.add_(1)
            q = R.paged_append(qkv[i], k, v, table, n, None, None, H, status=status)
            pause()
            ys.append(R.paged_attn_decode_shared(q.view(B, H, D), k, v, table, n, starts, shared, workspace=ws, status=status))
            pause()
        return torch.stack(ys)

    want = run(torch.cuda.synchronize)
    graph = torch.cuda.CUDAGraph()
    if captured:
        with torch.cuda.graph(graph):
            ys = run(lambda: None)
    for _ in range(5):
        for x, old in zip((k, v, n), keep):
            x.copy_(old)
        if captured:
            ys.zero_()
            graph.replay()
        else:
            ys = run(lambda: None)
        assert torch.equal(ys, want) and int(status) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("bf16", "bf16")])
def test_prompt_rows_that_a_block_took_are_nan(io, cache):
    """The same of qd_paged_attn_prompt: 700 prompts of 20 rows, of which block 0 holds the last and another one."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    B, new = 700, 20
    k, v, table, n = make_cache(torch, [300] * B, 64, 1, cache)
    starts = torch.arange(B + 1, dtype=torch.int32, device="cuda") * new
    q = torch.randn(B * new, 4, D, device="cuda").to(_types(torch)[io])
    want = R.paged_attn_prompt(q, k, v, table, n, starts)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert _lib.load().qd_paged_inject_stall_at(_lib.QD_PAGED_STALL_LAST) == _lib.QD_OK
    y = R.paged_attn_prompt(q, k, v, table, n, starts, status=status)
    gone = y.isnan().any(-1).view(B, new * 4)
    assert int(status) == _lib.QD_PAGED_TIMEOUT and torch.equal(gone.any(-1), gone.all(-1))
    assert bool(gone[-1].all()) and int(gone.any(-1).sum()) == 2
    keep = ~gone.view(-1, 4)
    assert torch.equal(y[keep], want[keep]) and bool(y[~keep].isnan().all())
    status.zero_()
    assert torch.equal(R.paged_attn_prompt(q, k, v, table, n, starts, status=status), want) and int(status) == 0


@pytest.mark.gpu
def test_calls_on_several_streams_at_once():
    """Five streams with calls of their own, none waiting for another: every result is the one of the call alone."""
    torch = _cuda()
    from kernel_optimization_webgpu_b200 import runtime as R
    work = []
    for i, (sizes, prefix, heads, io) in enumerate([([40], [3000], 8, "f16"), ([2] * 60, [200 + i for i in range(60)], 8, "f32"),
                                                    ([1], [50], 2, "f16"), ([9, 1, 30], [700, 0, 1500], 16, "f32"), ([5], [129], 4, "f16")]):
        c = make_shared(torch, sizes, prefix, [1 + 7 * b % 90 for b in range(sum(sizes))], 32, 2, "f16", seed=i)
        work.append((torch.randn(sum(sizes), heads, D, device="cuda").to(_types(torch)[io]), *c[:6]))
    want = [R.paged_attn_decode_shared(*w) for w in work]
    streams = [torch.cuda.Stream() for _ in work]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    got = [[] for _ in work]
    for _ in range(30):
        for i, s in enumerate(streams):
            got[i].append(R.paged_attn_decode_shared(*work[i], status=status, stream=s))
    torch.cuda.synchronize()
    assert int(status) == 0
    for ys, y in zip(got, want):
        assert all(torch.equal(x, y) for x in ys)
