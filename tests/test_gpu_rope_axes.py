"""GPU: rotary positions with several axes (ops.rope_axes, rope_axes_cache_write, rope_remap_axes) against the formula in
64 bits.

Tolerance, element by element: half a step of the type (the one rounding of the result), and of fp32 work 2^-21 of
|x1| + |x2|: cos and sin are off by at most 2^-22 (the angle's fraction rounded to fp32, half an ulp of half a turn =
2^-25 turns = 2^-22.3 radians, and two ulps of the function, 2^-23), the product and sum by 2^-23 of |x1| + |x2|."""
import pytest
import torch

from tests.inputs import gen, randn, randperm

pytestmark = pytest.mark.gpu

DT = [torch.bfloat16, torch.float16, torch.float32]


def axis_map(sections, interleaved):
    n, half = len(sections), sum(sections)
    if not interleaved:
        return [a for a, c in enumerate(sections) for _ in range(c)]
    return [j % n if j < n * sections[j % n] else 0 for j in range(half)]


def inv_freq(half, theta, dev):
    return (1.0 / theta ** (torch.arange(half, dtype=torch.float32) / half)).to(dev)


def rotate64(x, pos, inv, sections, interleaved=False, adjacent=False, inverse=False):
    """(result in 64 bits, tolerance) of x [T, H, D] at pos [A, T]."""
    half = inv.numel()
    ang = (pos.double()[axis_map(sections, interleaved)] * inv.double()[:, None]).t()[:, None]  # [T, 1, half]
    c, s = torch.cos(ang), torch.sin(ang) * (-1 if inverse else 1)
    y = x.double().clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if adjacent else (slice(0, half), slice(half, 2 * half))
    x1, x2 = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = x1 * c - x2 * s, x1 * s + x2 * c
    tol = torch.zeros_like(y)
    size = x1.abs() + x2.abs()
    tol[..., a] = tol[..., b] = size * 2.0 ** -21
    tol += torch.finfo(x.dtype).eps / 2 * (y.abs() + tol) + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    tol[..., 2 * half:] = 0
    return y, tol


def check(got, ref, what=""):
    y, tol = ref
    bad = (got.double() - y).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got.double() - y).abs() - tol).max().item():.3e} over"


def positions(dev, axes, t, far, seed, dtype=torch.int32):
    return torch.randint(0, far, (axes, t), generator=gen(dev, seed), device=dev).to(dtype)


SHAPES = [  # hq, hkv, d, R, sections, interleaved, adjacent
    (32, 8, 128, 128, (16, 24, 24), False, False), (32, 8, 128, 128, (24, 20, 20), True, False), (16, 16, 64, 64, (16, 16), False, True),
    (24, 8, 128, 64, (11, 11, 10), False, False), (12, 12, 64, 32, (6, 5, 5), True, True), (8, 1, 256, 256, (128,), False, False),
    (3, 1, 80, 80, (10, 10, 10, 10), False, False), (5, 5, 72, 72, (0, 18, 18), False, True), (2, 2, 128, 2, (1,), False, False),
    (7, 7, 96, 48, (24,), False, True), (1, 1, 2, 2, (0, 1), False, False), (4, 2, 40, 20, (5, 5), True, False),
]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("t", [1, 2, 3, 37])
def test_rotation(dev, dtype, shape, t):
    from kessie_amd import ops
    hq, hkv, d, r, sections, inter, adj = shape
    inv = inv_freq(r // 2, 500000.0, dev)
    pos = positions(dev, len(sections), t, 1_000_000, 1)
    qkv = randn((t, hq + 2 * hkv, d), dtype, dev, 2)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hkv]
    want_q, want_k = (rotate64(x, pos, inv, sections, inter, adj) for x in (q, k))
    before = qkv.clone()
    qo, ko = torch.full((t, hq, d), float("nan"), dtype=dtype, device=dev), torch.full((t, hkv, d), float("nan"), dtype=dtype, device=dev)
    got = ops.rope_axes(q, k, pos, inv, sections, inter, adj, q_out=qo, k_out=ko)
    assert got[0] is qo and got[1] is ko and torch.equal(qkv, before)
    check(qo, want_q, "q")
    check(ko, want_k, "k")
    # In place, the same bits, and nothing else of the projection touched.
    ops.rope_axes(q, k, pos.long(), inv, sections, inter, adj)
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(qkv[:, hq + hkv:], before[:, hq + hkv:])
    # The inverse, of the rounded result.
    back = rotate64(qo, pos, inv, sections, inter, adj, inverse=True)
    ops.rope_axes(qo, None, pos, inv, sections, inter, adj, inverse=True)
    check(qo, back, "inverse")


def test_one_row_of_positions_is_every_axis(dev):
    from kessie_amd import ops
    q = randn((50, 4, 128), torch.bfloat16, dev, 0)
    inv, pos = inv_freq(64, 1e4, dev), positions(dev, 1, 50, 9000, 3)[0]
    a, _ = ops.rope_axes(q, None, pos, inv, (16, 24, 24), q_out=torch.empty_like(q))
    b, _ = ops.rope_axes(q, None, pos.expand(3, 50).contiguous(), inv, (16, 24, 24), q_out=torch.empty_like(q))
    c, _ = ops.rope_axes(q, None, pos, inv, (64,), q_out=torch.empty_like(q))
    assert torch.equal(a, b) and torch.equal(a, c)
    check(a, rotate64(q, pos[None], inv, (64,)))


@pytest.mark.parametrize("far", [2 ** 24 + 3, 2 ** 31 - 1, -(2 ** 31), 2 ** 40 + 12345])
def test_far_positions(dev, far):
    """Positions past 2^24 keep their angle (at 2^40, as far as 64 bits hold it: 2^40 / 2pi turns in 53 bits, 2^-15)."""
    from kessie_amd import ops
    q = randn((1, 2, 64), torch.float32, dev, 0)
    inv = inv_freq(32, 1e4, dev)
    pos = torch.full((1, 1), far, dtype=torch.int64 if abs(far) > 2 ** 31 else torch.int32, device=dev)
    got, _ = ops.rope_axes(q, None, pos, inv, (32,), q_out=torch.empty_like(q))
    y, tol = rotate64(q, pos, inv, (32,))
    # The turns are rounded twice in 64 bits: their error, in radians, per unit of |x1| + |x2|.
    size = q.double().abs()
    size = (size[..., :32] + size[..., 32:]).repeat(1, 1, 2)
    check(got, (y, tol + 4 * 2.0 ** -53 * abs(far) * size))


@pytest.mark.parametrize("layout", ["native", "kv_first", "block_kv"])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("t,p,shape", [(1, 16, SHAPES[0]), (70, 16, SHAPES[1]), (33, 32, SHAPES[3]), (19, 5, SHAPES[6]), (40, 16, SHAPES[2])])
def test_write(dev, layout, dtype, t, p, shape):
    from kessie_amd import ops
    hq, hkv, d, r, sections, inter, adj = shape
    n = -(-t // p) + 4
    lay = {"native": (n, p, 2, hkv, d), "kv_first": (2, n, p, hkv, d), "block_kv": (n, 2, p, hkv, d)}[layout]
    pool = randn(lay, dtype, dev, 5)
    order = {"native": (0, 1, 2, 3, 4), "kv_first": (1, 2, 0, 3, 4), "block_kv": (0, 2, 1, 3, 4)}[layout]
    before = pool.clone().permute(order)
    qkv = randn((t, hq + 2 * hkv, d), dtype, dev, 6)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    slots = torch.randperm(n * p, generator=gen(dev, 7), device=dev)[:t].contiguous()
    slots[1::5] = -1
    if t > 10:
        slots[3] = n * p + 2  # outside the pool
    pos = positions(dev, len(sections), t, 100_000, 8)
    inv = inv_freq(r // 2, 1e4, dev)
    kv0 = qkv[:, hq:].clone()
    want_q, want_k = rotate64(q, pos, inv, sections, inter, adj), rotate64(k, pos, inv, sections, inter, adj)
    ops.rope_axes_cache_write(q, k, v, pos, pool, slots, inv, sections, inter, adj, layout=layout)
    check(q, want_q, "q")
    assert torch.equal(qkv[:, hq:], kv0)
    got = pool.permute(order)
    live = (slots >= 0) & (slots < n * p)
    pg, at = slots[live] // p, slots[live] % p
    check(got[pg, at, 0], (want_k[0][live], want_k[1][live]), "k")
    assert torch.equal(got[pg, at, 1], v[live])
    rest = torch.ones(n, p, dtype=torch.bool, device=dev)
    rest[pg, at] = False
    assert torch.equal(got[rest], before[rest])
    # Without Q, the same cache; and the same K as rope_axes followed by kv_cache_write.
    again, two = before.clone().contiguous(), before.clone().contiguous()
    ops.rope_axes_cache_write(None, k, v, pos, again, slots, inv, sections, inter, adj)
    ops.kv_cache_write(two, ops.rope_axes(k, None, pos, inv, sections, inter, adj, q_out=torch.empty(t, hkv, d, dtype=dtype, device=dev))[0],
                       v, slots)
    assert torch.equal(again, got) and torch.equal(two, got)


@pytest.mark.parametrize("layout", ["native", "kv_first", "dense"])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("t,shape", [(1, SHAPES[0]), (100, SHAPES[0]), (531, SHAPES[1]), (45, SHAPES[3]), (64, SHAPES[2]), (31, SHAPES[6])])
def test_remap(dev, layout, dtype, t, shape):
    from kessie_amd import ops
    _, h, d, r, sections, inter, adj = shape
    p, n = 16, -(-t // 16) + 3
    inv = inv_freq(r // 2, 500000.0, dev)
    a, b = positions(dev, len(sections), t, 1_000_000, 3), positions(dev, len(sections), t, 1_000_000, 4)
    if layout == "dense":
        k = randn((t, h, d), dtype, dev, 1)
        want = rotate64(k, b.long() - a, inv, sections, inter, adj)
        ops.rope_remap_axes(k, a, b, inv, sections, inter, adj)
        check(k, want)
        return
    pool = randn((n, p, 2, h, d) if layout == "native" else (2, n, p, h, d), dtype, dev, 1)
    pages = randperm(n, dev, 2)[:-(-t // p)].contiguous()
    if t > 40:
        pages[1] = n + 7  # no such page: left alone
    view = pool if layout == "native" else pool.permute(1, 2, 0, 3, 4)
    before = view.clone()
    tok = torch.arange(t, device=dev)
    pg, at = pages.long()[tok // p], tok % p
    live = pg < n
    pg, at = pg[live], at[live]
    want = rotate64(view[pg, at, 0], (b.long() - a)[:, live], inv, sections, inter, adj)
    ops.rope_remap_axes(pool, a, b, inv, sections, inter, adj, page_list=pages, layout=layout)
    check(view[pg, at, 0], want)
    assert torch.equal(view[:, :, 1], before[:, :, 1])
    rest = torch.ones(n, p, dtype=torch.bool, device=dev)
    rest[pg, at] = False
    assert torch.equal(view[rest], before[rest])


def test_equal_axes_remap_as_the_single_axis(dev):
    """Axes that move alike: within two roundings of the one-axis remap (its angle is an fp32 product: small positions)."""
    from kessie_amd import ops
    k = randn((200, 8, 128), torch.float32, dev, 1)
    a, b = positions(dev, 1, 200, 64, 3)[0], positions(dev, 1, 200, 64, 4)[0]
    one = k.clone()
    ops.rope_remap_paged(one, a, b, 10000.0)
    ops.rope_remap_axes(k, a, b, ops.inv_freq_table(128, 10000.0, dev), (16, 24, 24))
    # |delta| < 64: its fp32 product is off by 64 * 2^-24 radians at most.
    assert (one - k).abs().max() <= (64 * 2.0 ** -24 + 2.0 ** -21) * 2 * one.abs().max()


@pytest.mark.parametrize("offset", [1, 2])
def test_rows_that_are_not_16_byte_aligned(dev, offset):
    from kessie_amd import ops
    buf = randn((20 * 5 * 64 + 8,), torch.bfloat16, dev, 0)
    q = buf[offset:offset + 20 * 5 * 64].view(20, 5, 64)
    pos, inv = positions(dev, 2, 20, 5000, 1), inv_freq(32, 1e4, dev)
    want = rotate64(q, pos, inv, (16, 16))
    ops.rope_axes(q, None, pos, inv, (16, 16))
    check(q, want)


@pytest.mark.parametrize("t", [1, 37])
def test_head_major_rows(dev, t):
    """Tensors [H, T, D] seen as [T, H, D]: as inputs, outputs, and rotated in place."""
    from kessie_amd import ops
    pos, back, inv = positions(dev, 2, t, 5000, 1), positions(dev, 2, t, 5000, 2), inv_freq(32, 1e4, dev)
    q = randn((6, t, 64), torch.float16, dev, 3).transpose(0, 1)
    out = torch.zeros(6, t, 64, dtype=torch.float16, device=dev).transpose(0, 1)
    ops.rope_axes(q, None, pos, inv, (16, 16), q_out=out)
    check(out, rotate64(q, pos, inv, (16, 16)))
    want = rotate64(out, back.long() - pos, inv, (16, 16))
    ops.rope_remap_axes(out, pos, back, inv, (16, 16))
    check(out, want)


def test_more_tokens_than_one_grid_dimension(dev):
    from kessie_amd import ops
    t = (1 << 22) + 5
    q, pos, inv = randn((t, 1, 16), torch.bfloat16, dev, 3), positions(dev, 2, t, 1_000_000, 1), inv_freq(8, 1e4, dev)
    want = rotate64(q, pos, inv, (4, 4))
    ops.rope_axes(q, None, pos, inv, (4, 4))
    check(q, want)


def test_large_rows_past_32_bit_offsets(dev):
    """Token rows whose elements lie past 2^31: 70,000 tokens 32,768 elements apart (a 4.3 GiB projection)."""
    from kessie_amd import ops
    t, width = 70_000, 32_768
    big = torch.empty(t * width, dtype=torch.bfloat16, device=dev)
    q = big.view(t, width)[:, :2 * 128].view(t, 2, 128)
    q.copy_(randn((t, 2, 128), torch.bfloat16, dev, 3))
    pos, inv = positions(dev, 3, t, 100_000, 1), inv_freq(64, 1e4, dev)
    want = rotate64(q, pos, inv, (16, 24, 24))
    ops.rope_axes(q, None, pos, inv, (16, 24, 24))
    check(q, want)


def test_another_stream(dev):
    from kessie_amd import ops
    q, pos, inv = randn((300, 8, 128), torch.bfloat16, dev, 0), positions(dev, 3, 300, 5000, 1), inv_freq(64, 1e4, dev)
    want = ops.rope_axes(q, None, pos, inv, (16, 24, 24), q_out=torch.empty_like(q))[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(q)
    s.wait_stream(torch.cuda.current_stream())
    ops.rope_axes(q, None, pos, inv, (16, 24, 24), q_out=out, stream=s)
    s.synchronize()
    assert torch.equal(out, want)


def test_kernels_class(dev):
    from kessie_amd import ops
    from kessie_amd.kessie_hip_ctypes import KeSSieKernels
    k = KeSSieKernels()
    a, b, inv = positions(dev, 3, 70, 5000, 1), positions(dev, 3, 70, 5000, 2), inv_freq(64, 1e4, dev)
    pages = randperm(9, dev, 3)[:5].contiguous()
    pool = randn((9, 16, 2, 2, 128), torch.bfloat16, dev, 4)
    want, got = pool.clone(), [pool.clone(), pool.clone()]
    ops.rope_remap_axes(want, a, b, inv, (16, 24, 24), page_list=pages)
    k.rope_remap_axes(got[0], pages, a, b, inv, (16, 24, 24))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    k.rope_remap_axes(got[1], pages, a, b, inv, (16, 24, 24), stream=s)
    s.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], want) and not torch.equal(want, pool)
    dense = randn((70, 2, 128), torch.bfloat16, dev, 5)
    ref = rotate64(dense, b.long() - a, inv, (16, 24, 24))
    k.rope_remap_axes(dense, None, a, b, inv, (16, 24, 24))
    check(dense, ref)
    with pytest.raises(TypeError):
        k.rope_remap_axes(pool, pages.long(), a, b, inv, (16, 24, 24))
