"""Rotary positions of rows (lib.rotary) and the append to the paged cache (lib.rotary_kv_append) against float64: both pairings, whole and partial heads, odd sizes,
rows on no 16-byte boundary, far positions, rows without a place."""
import math

import pytest
import torch

from omchat_b200 import lib

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _turns(rot, theta=1e4, stretch=1.0):
    return torch.tensor([theta ** (-2.0 * i / max(rot, 1)) / (2 * math.pi * stretch) for i in range(rot // 2)], dtype=torch.float64)


def _exact(x, pos, turns, halves, m=1.0, back=False):
    """x [T, heads, head] -> its rotation in 64 bits, and |u| + |v| of the pair of every element (0 where nothing is rotated)."""
    x, r = x.double(), 2 * turns.numel()
    a = (pos.double()[:, None] * turns.to(x.device)).frac() * (-2 * math.pi if back else 2 * math.pi)
    c, s = (m * a.cos())[:, None], (m * a.sin())[:, None]
    y, size = x.clone(), torch.zeros_like(x)
    iu = torch.arange(r // 2, device=x.device) if halves else 2 * torch.arange(r // 2, device=x.device)
    iv = iu + (r // 2 if halves else 1)
    u, v = x[..., iu], x[..., iv]
    y[..., iu], y[..., iv] = u * c - v * s, v * c + u * s
    size[..., iu] = size[..., iv] = u.abs() + v.abs()
    return y, size


def _check(y, exact, size, m=1.0):
    # the angle to half a step of 2^-24 turns, sine and cosine to two steps, three roundings of products: less than four times 2^-23 of |u| + |v|; then the
    # result's own rounding
    bound = torch.finfo(y.dtype).eps / 2 * exact.abs() * 1.001 + m * size * 2.0 ** -21 + 1e-37
    off = (y.double() - exact).abs()
    assert (off <= bound).all(), (off - bound).max()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("halves", [True, False])
@pytest.mark.parametrize("T,heads,head,rot,pad", [(1, 32, 128, 128, 0), (1, 1, 2, 2, 0), (3, 5, 64, 32, 0), (77, 7, 64, 24, 1), (130, 3, 80, 80, 8), (33, 2, 20, 10, 0),
                                                  (9, 4, 128, 0, 0), (2000, 9, 128, 128, 0), (1201, 6, 256, 192, 16), (5, 3, 96, 48, 3)])
def test_rows(T, heads, head, rot, pad, halves, dtype):
    g = torch.Generator().manual_seed(T * 31 + rot)
    wide = torch.randn(T, heads * head + pad, generator=g).to(dtype).cuda()
    x = wide[:, pad:] if pad % 2 else wide[:, :heads * head]        # an odd offset: no 16-byte boundary
    pos = torch.randint(0, 5000, (T,), generator=g, dtype=torch.int32).cuda()
    turns = _turns(rot).cuda()
    for back, m in ((False, 1.0), (True, 1.25)):
        exact, size = _exact(x.view(T, heads, head) if x.is_contiguous() else x.unflatten(1, (heads, head)), pos, turns, halves, m, back)
        y = lib.rotary(x, pos, turns, heads, head, halves=halves, back=back, mscale=m)
        _check(y.view(T, heads, head), exact, size, m)
        # into rows of another stride, and in place
        other = torch.full((T, heads * head + 8), 7.0, dtype=dtype, device="cuda")
        lib.rotary(x, pos, turns, heads, head, halves=halves, back=back, mscale=m, out=other[:, :heads * head])
        assert torch.equal(other[:, :heads * head], y) and bool((other[:, heads * head:] == 7).all())
        here = wide.clone()
        view = here[:, pad:] if pad % 2 else here[:, :heads * head]
        lib.rotary(view, pos, turns, heads, head, halves=halves, back=back, mscale=m, out=view)
        assert torch.equal(view, y)


@pytest.mark.parametrize("first", [0, 131072, 1 << 24, (1 << 31) - 64])
def test_far_positions(first):
    x = torch.randn(64, 2 * 128, generator=torch.Generator().manual_seed(1)).cuda()
    pos = (first + torch.arange(64)).to(torch.int32).cuda()
    turns = _turns(128, 1e6, 4.0).cuda()
    # 64 bits of position times frequency leave 2^31 2^-53 turns of error at most
    exact, size = _exact(x.view(64, 2, 128), pos, turns, True)
    _check(lib.rotary(x, pos, turns, 2, 128).view(64, 2, 128), exact, size)


def test_no_rows():
    x = torch.empty(0, 128, device="cuda")
    assert lib.rotary(x, torch.empty(0, dtype=torch.int32, device="cuda"), _turns(128).cuda(), 1, 128).shape == (0, 128)


def test_back_is_the_gradient_and_the_inverse():
    g = torch.Generator().manual_seed(5)
    x, w = (torch.randn(200, 3 * 64, generator=g).cuda() for _ in range(2))
    pos, turns = torch.arange(1000, 1200, dtype=torch.int32).cuda(), _turns(48).cuda()
    f = lambda z, m=1.5: lib.rotary(z, pos, turns, 3, 64, halves=False, mscale=m)  # noqa: E731
    grad = lib.rotary(w, pos, turns, 3, 64, halves=False, back=True, mscale=1.5)
    # <w, f(x)> is linear in x: its gradient from differences along directions; sums of 38400 products of fp32 results
    for seed in range(3):
        d = torch.randn(200, 3 * 64, generator=torch.Generator().manual_seed(seed)).cuda()
        diff = (w.double() * (f(x + d).double() - f(x - d).double())).sum() / 2
        size = (w.double().abs() * (x.double().abs() + d.double().abs()) * 4).sum()
        assert abs(diff - (grad.double() * d.double()).sum()) <= size * 2.0 ** -21
    back = lib.rotary(f(x, 1.0), pos, turns, 3, 64, halves=False, back=True)
    assert ((back - x).abs() <= 2.0 ** -20 * (x.unflatten(1, (-1, 2)).abs().sum(-1, keepdim=True).expand(-1, -1, 2).flatten(1) + 1)).all()


# ---------------------------------------------------------------------------------------------------------------- the append
def _cache(n_seq, ctx, hkv, page, head, g, spare=3):
    per = max(1, -(-ctx // page))
    order = torch.randperm(n_seq * per + spare, generator=g)[: n_seq * per].to(torch.int32).view(n_seq, per)
    pool = torch.randn(n_seq * per + spare, 2, hkv, page, head, generator=g).to(BF)
    return pool.cuda(), order.cuda()


@pytest.mark.parametrize("halves", [True, False])
@pytest.mark.parametrize("hq,hkv,head,rot,page,lens", [(28, 4, 128, 128, 64, [1] * 9), (14, 2, 64, 64, 16, [33, 1, 100]), (4, 4, 80, 20, 7, [50, 3]), (6, 1, 128, 64, 1, [5, 9]),
                                                       (7, 1, 128, 128, 24, [700]), (8, 8, 64, 24, 128, [3, 260, 1]), (3, 3, 34, 34, 5, [11])])
def test_append(hq, hkv, head, rot, page, lens, halves):
    g = torch.Generator().manual_seed(hq * 100 + page)
    T, W = sum(lens), (hq + 2 * hkv) * head
    pool, table = _cache(len(lens), max(lens) + 40, hkv, page, head, g)
    before = pool.clone()
    qkv = torch.randn(T, W, generator=g).to(BF).cuda()
    pos = torch.cat([torch.arange(n) + 40 - 3 * i for i, n in enumerate(lens)]).to(torch.int32).cuda()
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).to(torch.int32).cuda()
    turns = _turns(rot).cuda()
    q = lib.rotary_kv_append(qkv, pos, seq, turns, hq, pool, table, halves=halves, mscale=1.125)
    rows = qkv.view(T, -1, head)
    exact, size = _exact(rows[:, :hq + hkv], pos, turns, halves, 1.125)
    _check(q.view(T, hq, head), exact[:, :hq], size[:, :hq], 1.125)
    at, slot = table[seq.long(), (pos // page).long()].long(), (pos % page).long()
    _check(pool[at, 0, :, slot], exact[:, hq:], size[:, hq:], 1.125)
    assert torch.equal(pool[at, 1, :, slot], rows[:, hq + hkv:])
    written = torch.zeros(pool.shape[0], page, dtype=torch.bool, device="cuda")
    written[at, slot] = True
    kept = ~written[:, None, None, :, None].expand_as(pool)
    assert torch.equal(pool[kept], before[kept])
    # in place, and from rows of another stride
    pool2, wide = before.clone(), torch.zeros(T, W + 8, dtype=BF, device="cuda")
    wide[:, :W] = qkv
    lib.rotary_kv_append(wide[:, :W], pos, seq, turns, hq, pool2, table, halves=halves, mscale=1.125, q_out=wide[:, :hq * head])
    assert torch.equal(pool2, pool) and torch.equal(wide[:, :hq * head], q) and torch.equal(wide[:, hq * head:W], qkv[:, hq * head:])


def test_append_rows_without_a_place():
    """Sequences, positions and pages outside the table or the pool: such rows are rotated and not appended."""
    g = torch.Generator().manual_seed(3)
    hq, hkv, head, page = 4, 2, 64, 16
    pool, table = _cache(2, 64, hkv, page, head, g)
    table[1, 2], table[1, 3] = -1, pool.shape[0]
    before = pool.clone()
    seq = torch.tensor([0, -1, 2, 0, 0, 1, 1, 1], dtype=torch.int32).cuda()
    pos = torch.tensor([5, 6, 7, -1, 64, 32, 48, 31], dtype=torch.int32).cuda()
    qkv = torch.randn(8, (hq + 2 * hkv) * head, generator=g).to(BF).cuda()
    turns = _turns(head).cuda()
    q = lib.rotary_kv_append(qkv, pos, seq, turns, hq, pool, table)
    exact, size = _exact(qkv.view(8, -1, head)[:, :hq], pos, turns, True)
    _check(q.view(8, hq, head), exact, size)
    for t in (0, 7):
        at, slot = int(table[seq[t], pos[t] // page]), int(pos[t] % page)
        assert torch.equal(pool[at, 1, :, slot], qkv[t].view(-1, head)[hq + hkv:])
        pool[at, :, :, slot] = before[at, :, :, slot]
    assert torch.equal(pool, before)


def test_append_one_sequence_without_ids():
    g = torch.Generator().manual_seed(4)
    pool, table = _cache(1, 70, 1, 64, 128, g)
    qkv, pos, turns = torch.randn(5, 9 * 128, generator=g).to(BF).cuda(), torch.arange(62, 67, dtype=torch.int32).cuda(), _turns(128).cuda()
    a = pool.clone()
    qa = lib.rotary_kv_append(qkv, pos, None, turns, 7, a, table)
    qb = lib.rotary_kv_append(qkv, pos, torch.zeros(5, dtype=torch.int32).cuda(), turns, 7, pool, table)
    assert torch.equal(a, pool) and torch.equal(qa, qb)
