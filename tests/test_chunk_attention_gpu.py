"""Attention of a chunk of new tokens over the paged cache (lib.paged_attention) against float64: chunks of no, one and many tokens, contexts that end inside pages and
tiles, groups of query heads of any size, what lies behind a context or outside the pool, rows without keys."""
import pytest
import torch

from omchat_b200 import lib

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _inputs(new, ctx, hq, hkv, head, page, seed=0, poison=True, extra=0, peak=1.0):
    """q [T (+ extra), hq * head] as columns of wider rows; a pool whose rows behind the contexts, and pages of nobody, are NaN."""
    g = torch.Generator().manual_seed(seed + 17 * sum(ctx) + hq)
    per = max(1, -(-max(ctx) // page))
    n_pages = len(new) * per + 2
    table = torch.randperm(n_pages, generator=g)[: len(new) * per].to(torch.int32).view(len(new), per)
    pool = torch.randn(n_pages, 2, hkv, page, head, generator=g).to(BF)
    if poison:
        clean = pool.clone()
        pool.fill_(float("nan"))
        for s, c in enumerate(ctx):
            for i in range(-(-c // page)):
                r = min(page, c - i * page)
                pool[table[s, i], :, :, :r] = clean[table[s, i], :, :, :r]
    T = sum(new) + extra
    q = (torch.randn(T, (hq + 3) * head, generator=g) * peak).to(BF).cuda()[:, head:(hq + 1) * head]
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    return q, pool.cuda(), table.cuda(), cu, torch.tensor(ctx, dtype=torch.int32).cuda()


def _check(out, q, pool, table, new, ctx, hq, hkv, head, scale):
    first = 0
    for s, (n, c) in enumerate(zip(new, ctx)):
        if n == 0:
            continue
        if c == 0:
            assert not out[first:first + n].any()
            first += n
            continue
        k, v = pool[table[s].long()].double().permute(1, 2, 0, 3, 4).reshape(2, hkv, -1, head)[:, :, :c]
        rows = q[first:first + n].double().view(n, hkv, hq // hkv, head)
        seen = torch.arange(c, device="cuda")[None] <= (c - n + torch.arange(n, device="cuda"))[:, None]
        for g in range(hkv):
            x = rows[:, g].transpose(0, 1)                                          # [rep, n, head]
            score = (x @ k[g].T) * scale
            size = (x.abs() @ k[g].T.abs()).masked_fill(~seen, 0).amax(-1) * scale
            p = torch.softmax(score.masked_fill(~seen, -torch.inf), -1).nan_to_num(0)
            exact, mean = p @ v[g], p @ v[g].abs()
            # scores in fp32 (products of head terms, at most 2^-20 of the sum of their magnitudes), probabilities and the result rounded to bf16 (half a
            # step each, 2^-8), exponentials to 2^-14; all errors meet the mean of |v| under the probabilities
            bound = mean * (2.0 ** -7 * 1.01 + 2.0 ** -13 + 2 * size[..., None] * 2.0 ** -20) + 1e-30
            got = out[first:first + n].double().view(n, hkv, hq // hkv, head)[:, g].transpose(0, 1)
            off = (got - exact).abs()
            assert (off <= bound).all(), (s, g, (off - bound).max().item(), off.max().item())
        first += n


CASES = [  # new, ctx, hq, hkv, head, page
    ([1], [1], 28, 4, 128, 64), ([1], [130], 28, 4, 128, 64), ([1], [1087], 28, 4, 128, 64), ([1, 1, 1], [64, 65, 127], 7, 1, 128, 16),
    ([1] * 9, [1, 2, 100, 128, 129, 256, 257, 700, 1500], 14, 2, 128, 24), ([5], [5], 4, 4, 64, 16), ([0, 3, 1, 0], [7, 3, 500, 0], 6, 2, 64, 1),
    ([18], [18], 7, 1, 128, 64), ([19], [400], 7, 1, 128, 100), ([37], [37], 28, 4, 128, 64), ([300], [1000], 28, 4, 128, 64), ([128], [128], 1, 1, 128, 64),
    ([129], [257], 2, 2, 64, 64), ([64, 1, 200, 5], [64, 900, 333, 2000], 8, 2, 128, 64), ([3], [300], 160, 1, 64, 32), ([2, 7], [129, 640], 72, 2, 128, 8),
    ([513], [513], 5, 1, 64, 128), ([700, 20], [2200, 20], 28, 4, 128, 64), ([1] * 40, [50 * i + 1 for i in range(40)], 28, 4, 128, 64),
]


@pytest.mark.parametrize("new,ctx,hq,hkv,head,page", CASES)
def test_against_float64(new, ctx, hq, hkv, head, page):
    q, pool, table, cu, lens = _inputs(new, ctx, hq, hkv, head, page)
    scale = head ** -0.5
    out = lib.paged_attention(q, pool, table, cu, lens, max(new), max(ctx), hq, scale)
    _check(out, q, pool, table, new, ctx, hq, hkv, head, scale)
    # the same bits again, also into rows of another stride and with bounds above the lengths
    wide = torch.full((q.shape[0], (hq + 1) * head), 3.0, device="cuda", dtype=BF)
    lib.paged_attention(q, pool, table, cu, lens, max(new), max(ctx), hq, scale, out=wide[:, head:])
    assert torch.equal(wide[:, head:], out) and bool((wide[:, :head] == 3).all())
    more = lib.paged_attention(q, pool, table, cu, lens, max(new) + 70, max(ctx) + 900, hq, scale)
    _check(more, q, pool, table, new, ctx, hq, hkv, head, scale)


@pytest.mark.parametrize("n,c", [(1, 40000), (9, 20001), (260, 9000)])
def test_long_contexts(n, c):
    q, pool, table, cu, lens = _inputs([n], [c], 14, 2, 128, 64)
    out = lib.paged_attention(q, pool, table, cu, lens, n, c, 14, 0.088)
    _check(out, q, pool, table, [n], [c], 14, 2, 128, 0.088)


@pytest.mark.parametrize("peak", [30.0, 1e-3])
def test_scores_far_apart_and_all_alike(peak):
    """Maxima that grow along the keys by far more than an exponent's range, and none."""
    new, ctx = [40, 1], [700, 1200]
    q, pool, table, cu, lens = _inputs(new, ctx, 14, 2, 128, 64, peak=peak)
    order = torch.arange(1, 1 + pool.shape[0], device="cuda").view(-1, 1, 1, 1)
    pool[:, 0] *= (order / pool.shape[0]).to(BF)
    out = lib.paged_attention(q, pool, table, cu, lens, 40, 1200, 14, 0.3)
    _check(out, q, pool, table, new, ctx, 14, 2, 128, 0.3)


def test_rows_behind_the_last_sequence_and_without_keys():
    new, ctx = [6, 4], [4, 100]                 # the first two rows of the first sequence have no position
    q, pool, table, cu, lens = _inputs(new, ctx, 14, 2, 64, 16, extra=5)
    out = torch.full((15, 14 * 64), 9.0, device="cuda", dtype=BF)
    lib.paged_attention(q, pool, table, cu, lens, 6, 100, 14, 0.125, out=out)
    assert bool((out[10:] == 9).all()) and bool((out[:2] == 0).all())
    _check(out[2:], q[2:], pool, table, [4, 4], ctx, 14, 2, 64, 0.125)
    # more rows than max_new says are not computed, and no row beyond q is touched
    out.fill_(9)
    lib.paged_attention(q, pool, table, cu, lens, 3, 100, 14, 0.125, out=out)
    assert bool((out[3:6] == 9).all()) and bool((out[9:] == 9).all()) and bool((out[:2] == 0).all())


def test_pages_outside_the_pool_read_as_zeros():
    new, ctx, page = [3, 2], [150, 260], 16
    q, pool, table, cu, lens = _inputs(new, ctx, 14, 2, 128, page, poison=False)
    held = torch.cat([pool, torch.zeros_like(pool[:1])])
    good = table.clone()
    good[0, 2] = good[1, 0] = good[1, 16] = pool.shape[0]
    bad = table.clone()
    bad[0, 2], bad[1, 0], bad[1, 16] = -1, pool.shape[0], 2 ** 31 - 1
    a = lib.paged_attention(q, pool, bad, cu, lens, 3, 260, 14, 0.088)
    b = lib.paged_attention(q, held, good, cu, lens, 3, 260, 14, 0.088)
    assert torch.equal(a, b)
    _check(a, q, held, good, new, ctx, 14, 2, 128, 0.088)


def test_numbers_that_are_not_finite():
    """A key that is NaN reaches every row that sees it, and none of another sequence; behind a context it reaches nobody (all other tests)."""
    new, ctx = [2, 2], [300, 300]
    q, pool, table, cu, lens = _inputs(new, ctx, 14, 2, 128, 64)
    pool[table[0, 1].item(), 0, 0, 5] = float("nan")
    out = lib.paged_attention(q, pool, table, cu, lens, 2, 300, 14, 0.088).view(4, 14, 128)
    assert bool(out[:2, :7].isnan().all()) and bool(out[:2, 7:].isfinite().all()) and bool(out[2:].isfinite().all())


def test_replay_goes_by_the_lengths_of_the_replay():
    new, ctx = [3, 1, 2], [200, 90, 777]
    q, pool, table, cu, lens = _inputs([4, 4, 4], [400, 400, 1000], 14, 2, 128, 64)
    out = torch.empty(12, 14 * 128, device="cuda", dtype=BF)
    call = lambda: lib.paged_attention(q, pool, table, cu, lens, 4, 1000, 14, 0.088, out=out)  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for n, c in (([4, 4, 4], [400, 400, 1000]), (new, ctx), ([1, 0, 4], [1, 5, 4])):
        cu.copy_(torch.tensor([0] + n).cumsum(0))
        lens.copy_(torch.tensor(c))
        out.fill_(5)
        graph.replay()
        _check(out, q, pool, table, n, c, 14, 2, 128, 0.088)
        assert bool((out[sum(n):] == 5).all())


def test_pools_beyond_31_bits():
    """Pages whose rows lie behind 2^31 elements and 2^32 bytes of the pool, written and read."""
    hq, hkv, head, page, c = 14, 2, 128, 64, 9000
    n_pages = (1 << 31) // (2 * hkv * page * head) + 200
    pool = torch.empty(n_pages, 2, hkv, page, head, dtype=BF, device="cuda")
    per, g = -(-c // page), torch.Generator().manual_seed(2)
    table = (n_pages - 1 - torch.randperm(per, generator=g)).to(torch.int32).view(1, per).cuda()
    qkv = torch.randn(c, (hq + 2 * hkv) * head, generator=g).to(BF).cuda()
    pos, turns = torch.arange(c, dtype=torch.int32).cuda(), torch.rand(64, dtype=torch.float64, generator=g).cuda()
    q = lib.rotary_kv_append(qkv, pos, None, turns, hq, pool, table)
    for n in (1, 300):
        cu, lens = torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([c], dtype=torch.int32).cuda()
        out = lib.paged_attention(q[c - n:], pool, table, cu, lens, n, c, hq, 0.088)
        _check(out, q[c - n:], pool, table, [n], [c], hq, hkv, head, 0.088)
    at = table[0, (pos // page).long()].long()
    assert torch.equal(pool[at, 1, :, (pos % page).long()], qkv.view(c, -1, head)[:, hq + hkv:])


def test_many_sequences():
    """More sequences than a warp has lanes, most of them short or empty, and one long one in a later group."""
    new = [(i * 7) % 4 for i in range(150)]
    ctx = [n + (i * 13) % 200 for i, n in enumerate(new)]
    new[97], ctx[97] = 60, 3000
    q, pool, table, cu, lens = _inputs(new, ctx, 14, 2, 64, 16)
    out = lib.paged_attention(q, pool, table, cu, lens, 60, 3000, 14, 0.125)
    _check(out, q, pool, table, new, ctx, 14, 2, 64, 0.125)


FEW = [  # calls of few rows a sequence and head: blocks that clusters share, of any number of tiles, and the line that is cut
    ([1, 0, 1, 1], [0, 5, 1, 64], 14, 2, 128, 64), ([4, 2], [2, 90], 14, 2, 64, 16), ([1, 1], [3000, 200], 40, 40, 64, 16), ([5] * 8, [100 * i + 5 for i in range(8)], 14, 2, 64, 16),
    ([4, 1, 3], [700, 2000, 5], 28, 4, 128, 24), ([1] * 60 + [0] * 30 + [1] * 60, [(i * 37) % 3000 + 1 for i in range(150)], 14, 2, 128, 64),
    ([1] * 1100, [800 if i == 700 else i % 90 + 1 for i in range(1100)], 3, 1, 64, 64), ([1], [20000], 4, 4, 64, 64), ([2, 1], [16000, 9], 14, 2, 64, 128), ([1] * 70, [999] * 70, 16, 2, 128, 64),
    ([4] * 40, [(i * 53) % 700 + 4 for i in range(40)], 28, 4, 128, 64), ([6, 6], [400, 77], 8, 1, 64, 64), ([1], [1500], 48, 1, 64, 64), ([1] * 3, [64 * 8, 64 * 8 + 1, 64 * 7], 4, 1, 128, 32),
    ([5], [900], 14, 2, 64, 16), ([4], [1001], 28, 4, 128, 64), ([1] * 32, [16 * i + 9 for i in range(32)], 28, 4, 128, 64), ([2], [640], 12, 1, 64, 64), ([1], [2048], 2, 2, 64, 64),
]


@pytest.mark.parametrize("new,ctx,hq,hkv,head,page", FEW, ids=range(len(FEW)))
def test_few_rows(new, ctx, hq, hkv, head, page):
    q, pool, table, cu, lens = _inputs(new, ctx, hq, hkv, head, page, extra=2)
    out = torch.full((q.shape[0], hq * head), 5.0, device="cuda", dtype=BF)
    lib.paged_attention(q, pool, table, cu, lens, max(new), max(ctx), hq, head ** -0.5, out=out)
    _check(out, q, pool, table, new, ctx, hq, hkv, head, head ** -0.5)
    assert bool((out[sum(new):] == 5).all())
    again = lib.paged_attention(q, pool, table, cu, lens, max(new), max(ctx), hq, head ** -0.5)
    assert torch.equal(again[: sum(new)], out[: sum(new)])


def test_few_rows_whose_numbers_are_not_finite():
    """What no row sees stays out; a NaN among the keys of a token reaches its rows and, of the others, only rows of the same sequence and key/value head."""
    new, ctx = [1, 2, 1], [200, 700, 3000]
    q, pool, table, cu, lens = _inputs(new, ctx, 14, 2, 128, 64)
    want = lib.paged_attention(q, pool, table, cu, lens, 2, 3000, 14, 0.088)
    assert bool(want.isfinite().all())
    pool[table[1, 3].long(), 0, 1, 5] = float("nan")
    got = lib.paged_attention(q, pool, table, cu, lens, 2, 3000, 14, 0.088)
    assert bool(got[1:3, 7 * 128:].isnan().all()) and torch.equal(got[1:3, : 7 * 128], want[1:3, : 7 * 128])
    assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])


def test_queries_and_results_in_the_same_rows():
    q, pool, table, cu, lens = _inputs([300, 5], [1000, 2000], 14, 2, 128, 64)
    want = lib.paged_attention(q, pool, table, cu, lens, 300, 2000, 14, 0.088)
    assert torch.equal(lib.paged_attention(q, pool, table, cu, lens, 300, 2000, 14, 0.088, out=q), want) and torch.equal(q, want)


def test_refusals_of_the_wrapper():
    q, pool, table, cu, lens = _inputs([2, 3], [40, 50], 4, 2, 64, 16)
    call = lambda **kw: lib.paged_attention(*[kw.get(k, v) for k, v in dict(q=q, pool=pool, table=table, cu=cu, lens=lens).items()], 3, 50, kw.get("hq", 4), 0.1, out=kw.get("out"))  # noqa: E731
    call()
    for bad in (dict(q=q.float()), dict(q=q[:, :-64]), dict(pool=pool.half()), dict(pool=pool[:, :1]), dict(pool=pool.transpose(2, 3)), dict(table=table.long()), dict(table=table[0]),
                dict(cu=cu[:-1]), dict(cu=cu.long()), dict(lens=lens[:1]), dict(out=torch.empty(5, 256, device="cuda")), dict(hq=3), dict(q=q.cpu()),
                dict(out=torch.empty(5, 260, device="cuda", dtype=BF)[:, :256])):
        with pytest.raises(lib.OmcError):
            call(**bad)


def test_two_streams_at_once():
    cases = [_inputs([n], [c], 14, 2, 128, 64, seed=i) for i, (n, c) in enumerate([(3, 5000), (40, 3000)])]
    alone = [lib.paged_attention(*x, m, 5000, 14, 0.088) for x, m in zip(cases, (3, 40))]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(20):
        for i, x in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(lib.paged_attention(*x, (3, 40)[i], 5000, 14, 0.088))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in got[i])


def test_append_then_attend_is_a_prompt_in_portions():
    """A prompt whose rows are appended and looked through in portions of any size, against the whole prompt in 64 bits."""
    hq, hkv, head, page, n = 14, 2, 128, 16, 430
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(n, (hq + 2 * hkv) * head, generator=g).to(BF).cuda()
    turns = (torch.tensor([1e6 ** (-2.0 * i / head) for i in range(head // 2)], dtype=torch.float64) / 6.283185307179586).cuda()
    per = -(-n // page)
    pool = torch.full((per + 1, 2, hkv, page, head), float("nan"), dtype=BF, device="cuda")
    table = torch.randperm(per + 1, generator=g)[:per].to(torch.int32).view(1, per).cuda()
    pos = torch.arange(n, dtype=torch.int32).cuda()
    q, out, first = torch.empty(n, hq * head, dtype=BF, device="cuda"), torch.empty(n, hq * head, dtype=BF, device="cuda"), 0
    for m in (1, 130, 7, 1, 256, 35):
        rows = slice(first, first + m)
        lib.rotary_kv_append(qkv[rows], pos[rows], None, turns, hq, pool, table, q_out=q[rows])
        cu, lens = torch.tensor([0, m], dtype=torch.int32).cuda(), torch.tensor([first + m], dtype=torch.int32).cuda()
        lib.paged_attention(q[rows], pool, table, cu, lens, m, first + m, hq, head ** -0.5, out=out[rows])
        first += m
    assert first == n
    _check(out, q, pool, table, [n], [n], hq, hkv, head, head ** -0.5)


def _step(x, pos, turns, hq, pool, table, cu, lens, n, c):
    q = lib.rotary_kv_append(x, pos, None, turns, hq, pool, table)
    return lib.paged_attention(q, pool, table, cu, lens, n, c, hq, 0.088)


@pytest.mark.parametrize("n,c", [(1, 700), (3, 5000), (90, 900)])
def test_right_behind_who_writes(n, c):
    """The kernels may be launched while the one in front still runs: rows, positions, lengths and pages that it writes are those that they read."""
    hq, hkv = 14, 2
    q, pool, table, cu, lens = _inputs([n], [c], hq, hkv, 128, 64, poison=False)
    g = torch.Generator().manual_seed(n)
    rows = [torch.randn(n, (hq + 2 * hkv) * 128, generator=g).to(BF).cuda() for _ in range(6)]
    pos, turns = torch.arange(c - n, c, dtype=torch.int32).cuda(), torch.rand(64, dtype=torch.float64, generator=g).cuda()
    want = []
    for x in rows:
        want.append(_step(x, pos, turns, hq, pool, table, cu, lens, n, c).clone())
        torch.cuda.synchronize()
    slow, x, now, len_ = torch.randn(4096, 4096, device="cuda"), torch.empty_like(rows[0]), torch.zeros_like(pos), torch.zeros_like(lens)
    got = []
    for r in rows * 3:
        slow = slow @ slow * 1e-3
        x.copy_(r)
        now.copy_(pos)
        len_.copy_(lens)
        got.append(_step(x, now, turns, hq, pool, table, cu, len_, n, c))
        for t in (x, now, len_):
            t.zero_()                                        # behind it: what they read must have been read
    for a, b in zip(got, want * 3):
        assert torch.equal(a, b)


def test_a_graph_in_which_streams_meet():
    hq, hkv, n, c = 14, 2, 2, 3000
    q, pool, table, cu, lens = _inputs([n], [c], hq, hkv, 128, 64, poison=False)
    x = torch.randn(n, (hq + 2 * hkv) * 128, generator=torch.Generator().manual_seed(3)).to(BF).cuda()
    pos, turns = torch.arange(c - n, c, dtype=torch.int32).cuda(), torch.rand(64, dtype=torch.float64).cuda()
    want = _step(x, pos, turns, hq, pool, table, cu, lens, n, c).clone()
    side, graph, other = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.zeros(1000, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            first = lib.rotary(x, pos, turns, hq + 2 * hkv, 128)
        other += 1
        main.wait_stream(side)
        second = _step(x, pos, turns, hq, pool, table, cu, lens, n, c)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            third = _step(x, pos, turns, hq, pool, table, cu, lens, n, c)
        main.wait_stream(side)
    for _ in range(3):
        graph.replay()
    assert torch.equal(second, want) and torch.equal(third, want) and torch.equal(first, lib.rotary(x, pos, turns, hq + 2 * hkv, 128)) and bool((other == 3).all())
