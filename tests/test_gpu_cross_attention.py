"""GPU: cross attention (ops.cross_attention) against the formula in 64 bits.

Tolerance, element by element, with A = sum_j p_j |v_j| (p the 64-bit probabilities), h half a step of the type and X the
largest sum_d |q_d k_d| * sm_scale of the row's keys:
  h |o|               the one rounding of the result
  2 h A               probabilities that enter the product rounded to the type (16-bit types; a numerator and its sum)
  2 X (D + 4) 2^-24 A scores summed in fp32 (D terms, each of at most one rounding, and the scaling), in numerator and sum
  2^-18 A             exp2 (2^-22), fp32 sums over keys in two or more partial sums (each of n terms of one sign, in blocks)
For fp32 h is 2^-24."""
import pytest
import torch

from tests.inputs import gen, randn

pytestmark = pytest.mark.gpu

DT = [torch.bfloat16, torch.float16, torch.float32]
FILL = 7.0


def ref64(q, k, v, seqs, kv_start, mask, scale):
    """(o, tolerance) in float64 for packed sequences of (queries, states)."""
    t, hq, d = q.shape
    hkv = k.shape[1]
    o, tol = torch.full(q.shape, FILL, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    h = torch.finfo(q.dtype).eps / 2
    at = 0
    for (c, n), s in zip(seqs, kv_start):
        rows = slice(at, at + c)
        at += c
        keep = torch.ones(n, dtype=torch.bool, device=q.device) if mask is None else mask[s:s + n].bool()
        o[rows] = 0
        if c == 0 or not bool(keep.any()):
            continue
        qq = q[rows].double().view(c, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
        kk, vv = (x[s:s + n][keep].double().permute(1, 0, 2).contiguous() for x in (k, v))
        x = torch.matmul(qq, kk.transpose(1, 2).contiguous()) * scale
        p = torch.softmax(x, -1)
        big = (torch.matmul(qq.abs(), kk.abs().transpose(1, 2).contiguous()) * abs(scale)).amax(-1, keepdim=True)
        y, a = torch.matmul(p, vv), torch.matmul(p, vv.abs())
        e = (h * y.abs() + (2 * h + 2 * big * (d + 4) * 2.0 ** -24 + 2.0 ** -18) * a) * (1 + 2.0 ** -7) + torch.finfo(q.dtype).smallest_normal * 2 * h
        for z, to in ((y, o), (e, tol)):
            to[rows] = z.view(hkv, hq // hkv, c, d).permute(2, 0, 1, 3).reshape(c, hq, d)
    return o, tol


def case(dev, seqs, hq, hkv, d, dtype, seed=0, extra_q=2, gap=0, masked=0.0, gain=1.0):
    tq = sum(c for c, _ in seqs)
    starts, at = [], gap
    for _, n in seqs:
        starts.append(at)
        at += n + gap
    q = randn((tq + extra_q, hq, d), dtype, dev, seed) * gain
    kv = randn((max(at, 1), 2, hkv, d), dtype, dev, seed + 1)
    mask = torch.rand(kv.shape[0], generator=gen(dev, seed + 2), device=dev) >= masked if masked else None
    i32 = dict(dtype=torch.int32, device=dev)
    qs = torch.tensor([0] + [sum(c for c, _ in seqs[:i + 1]) for i in range(len(seqs))], **i32)
    return dict(q=q, k=kv[:, 0] * gain, v=kv[:, 1], qs=qs, ks=torch.tensor(starts, **i32), kl=torch.tensor([n for _, n in seqs], **i32), mask=mask,
                seqs=seqs, starts=starts)


def attend(c, **kw):
    from kessie_amd import ops
    out = kw.pop("out", None)
    if out is None:
        out = torch.full(c["q"].shape, FILL, dtype=c["q"].dtype, device=c["q"].device)
    mq, mk = max([x for x, _ in c["seqs"]] + [0]), max([n for _, n in c["seqs"]] + [0])
    return ops.cross_attention(c["q"], c["k"], c["v"], c["qs"], kw.pop("mq", mq), c["ks"], c["kl"], kw.pop("mk", mk), key_mask=c["mask"], out=out,
                               **kw)


def check(c, got, scale=None):
    d = c["q"].shape[2]
    o, tol = ref64(c["q"], c["k"], c["v"], c["seqs"], c["starts"], c["mask"], d ** -0.5 if scale is None else scale)
    bad = ~((got.double() - o).abs() <= tol)
    if bad.any():
        w = bad.nonzero()[0].tolist()
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off, first at {w}: {got[tuple(w)].item()} for {o[tuple(w)].item()}, tolerance "
                             f"{tol[tuple(w)].item():.2e}; rows {sorted(set(bad.nonzero()[:, 0].tolist()))[:8]}")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (8, 2, 128), (32, 8, 128), (6, 2, 64), (16, 1, 128), (7, 1, 64), (40, 2, 128), (3, 3, 128)])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("q", [1, 5, 70])
def test_lengths(dev, dtype, hq, hkv, d, n, q):
    c = case(dev, [(q, n)], hq, hkv, d, dtype, seed=n + q)
    check(c, attend(c))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d", [2, 16, 40, 72, 80, 96, 112, 192, 256])
def test_other_head_dims(dev, dtype, d):
    c = case(dev, [(3, 70), (1, 5), (17, 130)], 4, 2, d, dtype, seed=d, masked=0.2)
    check(c, attend(c))


RAGGED = [(1, 700), (0, 90), (33, 0), (129, 64), (5, 1), (64, 1999), (1, 63), (300, 517), (2, 4096)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (32, 8, 128), (6, 2, 128), (16, 1, 64)])
@pytest.mark.parametrize("masked", [0.0, 0.3, 0.97])
def test_ragged_batches(dev, dtype, hq, hkv, d, masked):
    """Lengths of zero on both sides, gaps between the states, hidden states; rows behind the last sequence stay."""
    c = case(dev, RAGGED, hq, hkv, d, dtype, seed=3, gap=3, masked=masked)
    got = attend(c)
    check(c, got)
    assert torch.equal(got, attend(c))  # the same bits again


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("seqs,hq,hkv,d", [([(1, 1500)] * 20, 16, 16, 64), ([(1, 9000), (1, 3), (1, 20000)], 64, 8, 128),
                                           ([(4, 6001)], 32, 8, 128), ([(1, 30011)], 8, 1, 64), ([(2, 100)] * 300, 8, 8, 64),
                                           ([(1, 130)], 128, 8, 128)])
def test_few_queries_over_many_states(dev, dtype, seqs, hq, hkv, d):
    c = case(dev, seqs, hq, hkv, d, dtype, seed=5)
    check(c, attend(c))


@pytest.mark.parametrize("dtype", DT[:2])
@pytest.mark.parametrize("seqs,hq,hkv,d", [([(700, 2500), (257, 1001)], 32, 8, 128), ([(1000, 1500)] * 3, 8, 8, 64), ([(2000, 4003)], 16, 2, 128)])
def test_prompts(dev, dtype, seqs, hq, hkv, d):
    c = case(dev, seqs, hq, hkv, d, dtype, seed=6)
    check(c, attend(c))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("q", [1, 90])
def test_scales(dev, dtype, q):
    for scale in (1.0, 0.01, 0.0, -0.3):
        c = case(dev, [(q, 200), (q, 33)], 8, 2, 64, dtype, seed=8)
        check(c, attend(c, sm_scale=scale), scale)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("q", [1, 90])
def test_peaked_scores(dev, dtype, q):
    """Scores of hundreds: the largest key takes nearly all, wherever it comes (growing ones rescale at every step)."""
    for order in (0, 1, -1):
        c = case(dev, [(q, 777)], 8, 2, 128, dtype, seed=9, gain=4.0)
        if order:
            i = c["k"][:, 0, 0].float().argsort(descending=order < 0)
            c["k"], c["v"] = c["k"][i].contiguous(), c["v"][i].contiguous()
        check(c, attend(c))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("q", [1, 100])
def test_hidden_and_foreign_states_are_not_used(dev, dtype, d, q):
    """NaN and infinities in hidden states, in the gaps around a sequence's states and in a neighbour's."""
    c = case(dev, [(q, 100), (q, 37), (q, 64)], 8, 2, d, dtype, seed=11, gap=5, masked=0.4)
    c["mask"][c["starts"][1]:c["starts"][1] + 37] = False  # the second sequence sees nothing
    own = torch.zeros(c["k"].shape[0], dtype=torch.bool, device=dev)
    for s, (_, n) in zip(c["starts"], c["seqs"]):
        own[s:s + n] = True
    bad = ~(own & c["mask"])
    clean = attend(c)
    check(c, clean)
    at = c["starts"][1]
    assert (clean[q:2 * q] == 0).all()
    for value in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).max):
        k, v = c["k"].clone(), c["v"].clone()
        k[bad], v[bad] = value, value
        assert torch.equal(attend({**c, "k": k, "v": v}), clean), value
    # The mask as bytes, any of them not zero.
    assert torch.equal(attend({**c, "mask": c["mask"].to(torch.uint8) * 200}), clean)
    assert at > 0


@pytest.mark.parametrize("dtype", DT)
def test_infinite_values_come_through(dev, dtype):
    """An infinity or NaN in a state that is seen reaches its head_dim element, as in the formula."""
    for q in (1, 100):
        c = case(dev, [(q, 90)], 4, 2, 64, dtype, seed=12, extra_q=0)
        c["v"] = c["v"].clone()
        c["v"][7, 0, 3], c["v"][80, 1, 5] = float("inf"), float("nan")
        got = attend(c)
        assert (got[:, :2, 3] == float("inf")).all() and got[:, 2:, 5].isnan().all()
        c["v"][7, 0, 3] = c["v"][80, 1, 5] = 0
        got[:, :2, 3] = attend(c)[:, :2, 3]
        got[:, 2:, 5] = attend(c)[:, 2:, 5]
        check(c, got)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("q,n", [(1, 60), (1, 9000), (40, 60), (200, 4000)])
def test_nan_scores_come_through(dev, dtype, d, q, n):
    """A row whose scores are all NaN is NaN, and the rows beside it are as they were, also where the states are split; so is
    every row over a NaN key."""
    c = case(dev, [(q, n), (q, 50)], 8, 2, d, dtype, seed=15)
    want = attend(c)
    c["q"][q // 2, 3] = float("nan")
    got = attend(c)
    assert got[q // 2, 3].isnan().all()
    got[q // 2, 3] = want[q // 2, 3]
    assert torch.equal(got, want)
    c = case(dev, [(q, n), (q, 50)], 8, 2, d, dtype, seed=15)
    c["k"] = c["k"].clone()
    c["k"][n - 1, 1] = float("nan")
    got = attend(c)
    assert got[:q, 4:].isnan().all()
    got[:q, 4:] = want[:q, 4:]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("q", [1, 40])
def test_shared_overlapping_and_cut_ranges(dev, dtype, q):
    from kessie_amd import ops
    c = case(dev, [(q, 150)] * 5, 8, 2, 64, dtype, seed=13, extra_q=0)
    c["k"], c["v"] = c["k"][:400].contiguous(), c["v"][:400].contiguous()
    n = 400
    for starts, lens in [([0, 0, 100, 250, 399], [150, 150, 150, 150, 1]), ([-1, 400, 350, 0, 7], [10, 10, 150, -5, 1 << 30])]:
        c["ks"].copy_(torch.tensor(starts)), c["kl"].copy_(torch.tensor(lens))
        cut = [(0 if s < 0 or s >= n else max(0, min(x, 200, n - s))) for s, x in zip(starts, lens)]
        got = attend(c, mk=200)
        d = {**c, "seqs": [(q, x) for x in cut], "starts": [max(0, min(s, n)) for s in starts]}
        check(d, got)
    # Query offsets that do not start at zero (a slice of a longer batch's), and chunks cut at max_query_len.
    c = case(dev, [(q, 150)] * 3, 8, 2, 64, dtype, seed=14, extra_q=0)
    got = attend({**c, "qs": c["qs"] + 1000})
    check(c, got)
    if q > 1:
        out = attend(c, mq=q - 1)
        for b in range(3):
            assert torch.equal(out[b * q:(b + 1) * q - 1], got[b * q:(b + 1) * q - 1]) and (out[(b + 1) * q - 1] == FILL).all()
    # Offsets past the tensors are not followed.
    far = c["qs"].clone()
    far[3] = 1 << 30
    out = attend({**c, "qs": far})
    check(c, out)
    assert ops is not None


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("q", [1, 77])
def test_strides(dev, dtype, q):
    """Padded batches [B, L, H, D], head-major states [H, N, D], a strided output, rows that are not 16-byte aligned."""
    from kessie_amd import ops
    b, L, hq, hkv, d = 3, 91, 8, 2, 64
    i32 = dict(dtype=torch.int32, device=dev)
    lens = [91, 13, 60]
    qp = randn((b, q, hq, d), dtype, dev, 1)
    kp, vp = randn((b, L, hkv, d), dtype, dev, 2), randn((b, L, hkv, d), dtype, dev, 3)
    c = dict(q=qp.view(b * q, hq, d), k=kp.view(b * L, hkv, d), v=vp.view(b * L, hkv, d), mask=None, seqs=[(q, n) for n in lens],
             starts=[L * i for i in range(b)], qs=torch.arange(0, b * q + 1, q, **i32), ks=torch.arange(0, b * L, L, **i32),
             kl=torch.tensor(lens, **i32))
    plain = attend(c)
    check(c, plain)
    heads = kp.view(b * L, hkv, d).transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(attend({**c, "k": heads}), plain)
    wide = torch.full((b * q, hq + 3, 2 * d), FILL, dtype=dtype, device=dev)
    attend(c, out=wide[:, 1:hq + 1, d:])
    assert torch.equal(wide[:, 1:hq + 1, d:], plain)
    wide[:, 1:hq + 1, d:] = FILL
    assert (wide == FILL).all()
    for name in ("q", "k", "v"):
        odd = torch.empty(c[name].numel() + 1, dtype=dtype, device=dev)[1:].view(c[name].shape)
        odd.copy_(c[name])
        check(c, attend({**c, name: odd}))
    odd = torch.empty(plain.numel() + 1, dtype=dtype, device=dev)[1:].view(plain.shape)
    check(c, attend(c, out=odd))
    short = torch.zeros(c["k"].shape[0], hkv, d + 1, dtype=dtype, device=dev)  # rows of an odd length
    short[..., :d] = c["k"]
    check(c, attend({**c, "k": short[..., :d]}))
    assert ops is not None


@pytest.mark.parametrize("q", [1, 200])
def test_offsets_past_32_bits(dev, q):
    """States whose elements lie past 2^31: 40,000 rows of 65,536 elements (a 5.2 GB tensor), read at both ends."""
    n, width = 40_000, 65_536
    big = torch.empty(n * width, dtype=torch.bfloat16, device=dev)
    rows = big.view(n, width)
    k, v = rows[:, :2 * 64].view(n, 2, 64), rows[:, 2 * 64:4 * 64].view(n, 2, 64)
    k.copy_(randn((n, 2, 64), torch.bfloat16, dev, 1)), v.copy_(randn((n, 2, 64), torch.bfloat16, dev, 2))
    c = case(dev, [(q, 300), (q, 300), (q, 33_000)], 8, 2, 64, torch.bfloat16, seed=4)
    c.update(k=k, v=v, starts=[0, n - 300, 5000])
    c["ks"].copy_(torch.tensor(c["starts"]))
    check(c, attend(c))


@pytest.mark.parametrize("seqs", [[(1, 5000)] * 3, [(200, 3001)]])
def test_streams_and_own_workspaces(dev, seqs):
    """Two calls at once on two streams, each with its own workspace."""
    from kessie_amd import _lib
    a, b = case(dev, seqs, 32, 8, 128, torch.bfloat16, seed=1), case(dev, seqs, 32, 8, 128, torch.bfloat16, seed=2)
    want = [attend(a), attend(b)]
    t = a["q"].shape[0]
    need = _lib.load().kessie_cross_attention_workspace_bytes(len(seqs), seqs[0][0], t, a["k"].shape[0], 32, 8, 128, seqs[0][1], _lib.DTYPE_BF16)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    wss = [torch.empty(max(need, 1), dtype=torch.uint8, device=dev) for _ in streams]
    outs = [torch.zeros_like(a["q"]) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s, w, o in zip((a, b), streams, wss, outs):
            attend(c, stream=s, ws=w, out=o)
    torch.cuda.synchronize()
    for c, o, w in zip((a, b), outs, want):
        assert torch.equal(o[:sum(x for x, _ in seqs)], w[:sum(x for x, _ in seqs)])


def test_a_workspace_that_is_too_small_is_refused(dev):
    from kessie_amd import _lib
    c = case(dev, [(1, 60000)], 8, 1, 128, torch.bfloat16, seed=1)
    need = _lib.load().kessie_cross_attention_workspace_bytes(1, 1, c["q"].shape[0], 60000, 8, 1, 128, 60000, _lib.DTYPE_BF16)
    if need:
        out = torch.full_like(c["q"], FILL)
        with pytest.raises(_lib.KeSSieError) as e:
            attend(c, ws=torch.empty(need - 1, dtype=torch.uint8, device=dev), out=out)
        assert e.value.status == _lib.ERR_WORKSPACE and (out == FILL).all()


@pytest.mark.parametrize("q,n", [(1, 9000), (300, 2000)])
def test_captured_calls_follow_their_inputs(dev, q, n):
    """A graph of two calls (they share a workspace, in stream order), replayed with other inputs and lengths."""
    a, b = case(dev, [(q, n)] * 2, 16, 4, 128, torch.float16, seed=1), case(dev, [(q, n)] * 2, 16, 4, 128, torch.float16, seed=2)
    outs = [attend(a), attend(b)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        attend(a, out=outs[0])
        attend(b, out=outs[1])
    for i, lens in enumerate(([n, n], [n - 1, 0], [17, n // 2])):
        for c in (a, b):
            c["q"].copy_(randn(tuple(c["q"].shape), torch.float16, dev, 30 + i))
            c["kl"].copy_(torch.tensor(lens))
        for o in outs:
            o.fill_(FILL)
        g.replay()
        torch.cuda.synchronize()
        for c, o in zip((a, b), outs):
            check({**c, "seqs": [(q, x) for x in lens]}, o)
            assert torch.equal(o, attend(c))


def test_kernels_class(dev):
    from kessie_amd.kessie_hip_ctypes import KeSSieKernels
    c = case(dev, [(3, 40), (1, 7)], 8, 2, 64, torch.bfloat16, seed=1, extra_q=0)
    got = KeSSieKernels().cross_attention(c["q"], c["k"], c["v"], c["qs"], 3, c["ks"], c["kl"], 40)
    check(c, got)


@pytest.mark.parametrize("seqs,d", [([(1, 60), (1, 9000)], 64), ([(40, 60)] * 2, 128), ([(200, 4000), (3, 5)], 64), ([(700, 900)], 128),
                                    ([(30, 70)], 80)])
def test_in_place(dev, seqs, d):
    """out may be q."""
    c = case(dev, seqs, 8, 2, d, torch.bfloat16, seed=16, extra_q=0)
    want = attend(c)
    q = c["q"].clone()
    assert attend({**c, "q": q}, out=q) is q and torch.equal(q, want)


def test_testing_switches(dev, monkeypatch):
    """KESSIE_FORCE_GENERIC takes the generic kernel, KESSIE_REQUIRE_MFMA refuses what would."""
    from kessie_amd import _lib
    c = case(dev, [(3, 40), (200, 900)], 8, 2, 64, torch.bfloat16, seed=1)
    monkeypatch.setenv("KESSIE_REQUIRE_MFMA", "1")
    check(c, attend(c))
    out = torch.full_like(c["q"], FILL)
    odd = torch.empty(c["k"].numel() + 1, dtype=torch.bfloat16, device=dev)[1:].view(c["k"].shape)
    with pytest.raises(_lib.KeSSieError) as e:
        attend({**c, "k": odd}, out=out)
    assert e.value.status == _lib.ERR_UNSUPPORTED and (out == FILL).all()
    monkeypatch.setenv("KESSIE_FORCE_GENERIC", "1")
    with pytest.raises(_lib.KeSSieError):
        attend(c, out=out)
    monkeypatch.delenv("KESSIE_REQUIRE_MFMA")
    check(c, attend(c))


def test_many_sequences_and_a_long_one(dev):
    """20,000 sequences of no or few states around one whose rows are cut: every piece has a workgroup."""
    gen_ = torch.Generator().manual_seed(3)
    seqs = [(int(c), int(n)) for c, n in zip(torch.randint(0, 3, (20000,), generator=gen_), torch.randint(0, 4, (20000,), generator=gen_))]
    for at in (0, 12345, 19999):
        seqs[at] = (90, 40000)
    c = case(dev, seqs, 2, 1, 64, torch.bfloat16, seed=17)
    got = attend(c)
    assert torch.equal(got, attend(c))
    starts = [sum(x for x, _ in seqs[:i]) for i in (0, 12345, 19999)]
    for i, s in zip((0, 12345, 19999), starts):  # alone: the same rows within both roundings
        one = {**c, "q": c["q"][s:s + 90].contiguous(), "qs": torch.tensor([0, 90], dtype=torch.int32, device=dev), "ks": c["ks"][i:i + 1].contiguous(),
               "kl": c["kl"][i:i + 1].contiguous(), "seqs": [(90, 40000)], "starts": [c["starts"][i]]}
        check(one, got[s:s + 90])
    some = [i for i, (x, n) in enumerate(seqs[:300]) if x and i]
    for i in some[:40]:
        x, n = seqs[i]
        s = sum(y for y, _ in seqs[:i])
        check({**c, "q": c["q"][s:s + x].contiguous(), "seqs": [(x, n)], "starts": [c["starts"][i]]}, got[s:s + x])
