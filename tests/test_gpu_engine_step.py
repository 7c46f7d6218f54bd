"""GPU: steps of an engine made of its parts -- the step's tables (KeSSieAttentionMetadata.build), rotation into the cache,
paged attention, eviction, the remap that closes the gap, cross attention to encoder states -- each part checked on what the
part before it left, against plain bookkeeping on the host and 64-bit arithmetic; and a decode step captured in a graph."""
import pytest
import torch

from tests.exact64 import attend64, close_to_rounding
from tests.inputs import randn
from tests.test_gpu_cross_attention import ref64
from tests.test_gpu_rope_axes import inv_freq, rotate64

pytestmark = pytest.mark.gpu

HQ, HKV, D, P, PAGES, WIDTH = 8, 2, 64, 16, 40, 12
SECTIONS = (12, 10, 10)
STATES = [70, 0, 333]  # encoder states of each request


def three(positions):
    """Positions of three axes of tokens counted along the text: time, and a grid of 8 columns."""
    return torch.stack([positions, positions // 8, positions % 8]).to(torch.int32)


def within(got, ref):
    y, tol = ref
    assert ((got.double() - y).abs() <= tol).all()


class Engine:
    def __init__(self, dev):
        self.dev = dev
        self.inv = inv_freq(D // 2, 10000.0, dev)
        i32 = dict(dtype=torch.int32, device=dev)
        self.pool = randn((2, PAGES, P, HKV, D), torch.bfloat16, dev, 1)
        self.table = torch.full((3, WIDTH), -5, **i32)
        self.valid, self.where = torch.zeros(PAGES, dtype=torch.int8, device=dev), torch.zeros(PAGES, **i32)
        n = sum(STATES)
        self.ek, self.ev = randn((n, HKV, D), torch.bfloat16, dev, 2), randn((n, HKV, D), torch.bfloat16, dev, 3)
        self.starts = [0, STATES[0], STATES[0]]
        self.ks, self.kl = torch.tensor(self.starts, **i32), torch.tensor(STATES, **i32)
        # The host's books: of each request its tokens' (position, exact K, V), and its pages.
        self.k = [torch.zeros(0, HKV, D, dtype=torch.float64, device=dev) for _ in range(3)]
        self.ktol = [torch.zeros(0, HKV, D, dtype=torch.float64, device=dev) for _ in range(3)]
        self.v = [torch.zeros(0, HKV, D, dtype=torch.bfloat16, device=dev) for _ in range(3)]
        self.pages = [[], [], []]
        self.lens, self.delta = [0, 0, 0], [0, 0, 0]

    def rows(self, b):
        """Slots of request b's tokens, by the host's books."""
        at = torch.arange(self.lens[b], device=self.dev)
        return torch.tensor(self.pages[b] + [0], device=self.dev)[at // P], at % P

    def step(self, new, free, seed):
        from kessie_amd import ops
        from kessie_amd.kessie_attention import KeSSieAttentionImpl, KeSSieAttentionMetadata
        dev, tokens = self.dev, sum(new)
        qkv = randn((tokens, HQ + 2 * HKV, D), torch.bfloat16, dev, seed)
        q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]
        pool_before = self.pool.clone()
        meta = KeSSieAttentionMetadata.build(self.table, self.lens, new, P, free, position_delta=self.delta, page_valid=self.valid,
                                             page_positions=self.where)
        pos = three(meta.positions)
        q_rot = torch.empty(tokens, HQ, D, dtype=q.dtype, device=dev)
        ops.rope_axes_cache_write(q, k, v, pos, self.pool, meta.slot_mapping, self.inv, SECTIONS, q_out=q_rot, layout="kv_first")
        impl = KeSSieAttentionImpl(HQ, D, D ** -0.5, HKV)
        own = impl.forward(None, q_rot.view(tokens, -1), None, None, self.pool, meta).view(tokens, HQ, D)
        out = ops.cross_attention(own, self.ek, self.ev, meta.query_start_loc, meta.max_query_len, self.ks, self.kl, max(STATES))
        # The same by the books.
        at, takes = 0, free.tolist()
        written = torch.zeros(PAGES, P, dtype=torch.bool, device=dev)
        for b, n in enumerate(new):
            held = len(self.pages[b])
            while len(self.pages[b]) * P < self.lens[b] + n:
                self.pages[b].append(takes.pop(0))
            first = self.lens[b] + self.delta[b]
            self.lens[b] += n
            want = three(torch.arange(first, first + n, device=dev))
            assert torch.equal(pos[:, at:at + n], want)
            within(q_rot[at:at + n], rotate64(q[at:at + n], want, self.inv, SECTIONS))
            y, tol = rotate64(k[at:at + n], want, self.inv, SECTIONS)
            self.k[b], self.ktol[b], self.v[b] = torch.cat([self.k[b], y]), torch.cat([self.ktol[b], tol]), torch.cat([self.v[b], v[at:at + n]])
            pg, off = self.rows(b)
            written[pg[self.lens[b] - n:], off[self.lens[b] - n:]] = True
            for i in range(held, len(self.pages[b])):
                assert self.valid[self.pages[b][i]] == 1 and self.where[self.pages[b][i]] == i * P + self.delta[b]
            at += n
        assert meta.seq_lens.tolist() == self.lens and meta.pages_taken == free.numel() - len(takes)
        self.check_cache()
        assert torch.equal(self.pool[:, ~written], pool_before[:, ~written])
        at = 0
        for b, n in enumerate(new):
            pg, off = self.rows(b)
            ref = attend64(q_rot[at:at + n], self.pool[0, pg, off], self.pool[1, pg, off], self.lens[b] - n)
            close_to_rounding(own[at:at + n], ref, torch.bfloat16)
            at += n
        o, tol = ref64(own, self.ek, self.ev, list(zip(new, STATES)), self.starts, None, D ** -0.5)
        assert ((out.double() - o).abs() <= tol).all()
        return free[meta.pages_taken:].contiguous()

    def check_cache(self):
        for b in range(3):
            assert self.table[b, :len(self.pages[b])].tolist() == self.pages[b]
            pg, off = self.rows(b)
            within(self.pool[0, pg, off], (self.k[b], self.ktol[b]))
            assert torch.equal(self.pool[1, pg, off], self.v[b])

    def evict(self, before):
        """Pages that begin before position `before` go, of every request; their ids."""
        from kessie_amd import ops
        ids, count = ops.page_evict_list(self.valid, self.where, before)
        ids = ids[:int(count)]
        assert ids.tolist() == sorted(p for b in range(3) for i, p in enumerate(self.pages[b]) if i * P + self.delta[b] < before)
        for b in range(3):
            gone = sum(1 for i in range(len(self.pages[b])) if i * P + self.delta[b] < before)
            self.pages[b] = self.pages[b][gone:]
            self.table[b] = torch.cat([self.table[b, gone:], torch.full_like(self.table[b, :gone], -5)])
            cut = min(gone * P, self.lens[b])
            self.k[b], self.ktol[b], self.v[b] = self.k[b][cut:], self.ktol[b][cut:], self.v[b][cut:]
            self.lens[b] -= cut
            self.delta[b] += cut
        return ids

    def close_gap(self, b):
        """Request b's tokens are counted from zero again."""
        from kessie_amd import ops
        n, by = self.lens[b], self.delta[b]
        to = torch.arange(n, device=self.dev)
        old, new = three(to + by), three(to)
        ops.rope_remap_axes(self.pool, old, new, self.inv, SECTIONS, page_list=self.table[b, :len(self.pages[b])].contiguous(), layout="kv_first")
        # The exact K's rotation; the first rounding's error of both of a pair, the second rounding, and fp32's work.
        was = self.ktol[b].unflatten(-1, (2, D // 2)).sum(-2, keepdim=True).expand(-1, -1, 2, -1).flatten(-2)
        y = exact(self.k[b], new.long() - old, self.inv)
        h = torch.finfo(torch.bfloat16).eps / 2
        self.k[b], self.ktol[b] = y, was + h * (y.abs() + was) + 2.0 ** -20 * self.k[b].abs().amax()
        for i, p in enumerate(self.pages[b]):
            self.where[p] = i * P
        self.delta[b] = 0


def exact(k, pos, inv):
    axis = [a for a, c in enumerate(SECTIONS) for _ in range(c)]
    ang = (pos.double()[axis] * inv.double()[:, None]).t()[:, None]
    x1, x2 = k[..., :D // 2], k[..., D // 2:]
    return torch.cat([x1 * ang.cos() - x2 * ang.sin(), x1 * ang.sin() + x2 * ang.cos()], -1)


def test_steps_with_eviction_and_remap(dev):
    e = Engine(dev)
    free = torch.arange(PAGES - 1, -1, -1, dtype=torch.int32, device=dev)
    free = e.step([50, 35, 1], free, 10)          # prompts, and one of a single token
    free = e.step([1, 13, 70], free, 20)          # a chunk beside a decode
    free = e.step([1, 1, 1], free, 30)
    gone = e.evict(32)
    e.check_cache()
    e.close_gap(0)
    e.check_cache()
    free = torch.cat([gone, free])
    free = e.step([1, 1, 1], free, 40)            # positions count on where the gap stayed
    free = e.step([20, 1, 40], free, 50)
    assert e.lens[1] + e.delta[1] == 35 + 13 + 3 and e.delta == [0, 32, 32]


def test_a_captured_decode_step(dev):
    """Tables, rotation into the cache, decode and cross attention in one graph, replayed with the lengths and rows of other
    steps: what the eager calls give, bit for bit, and the same pages."""
    from kessie_amd import ops
    b, i32 = 3, dict(dtype=torch.int32, device=dev)
    inv = inv_freq(D // 2, 10000.0, dev)
    n = sum(STATES)
    ek, ev = randn((n, HKV, D), torch.bfloat16, dev, 2), randn((n, HKV, D), torch.bfloat16, dev, 3)
    ks, kl = torch.tensor([0, STATES[0], STATES[0]], **i32), torch.tensor(STATES, **i32)
    free = torch.arange(PAGES, **i32)

    def fresh():
        rows = dict(dtype=torch.bfloat16, device=dev)
        return dict(pool=randn((2, PAGES, P, HKV, D), torch.bfloat16, dev, 1), table=torch.arange(b * WIDTH, **i32).view(b, WIDTH),
                    have=torch.zeros(b, **i32), new=torch.ones(b, **i32), count=torch.zeros(1, **i32), free=free.clone(),
                    qkv=torch.zeros(b, HQ + 2 * HKV, D, **rows), q=torch.zeros(b, HQ, D, **rows), own=torch.zeros(b, HQ, D, **rows),
                    out=torch.zeros(b, HQ, D, **rows), tables=None)

    def step(s):
        s["tables"] = t = ops.step_tables(s["table"], s["have"], s["new"], P, b, s["free"], s["count"], out=s["tables"])
        q, k, v = s["qkv"][:, :HQ], s["qkv"][:, HQ:HQ + HKV], s["qkv"][:, HQ + HKV:]
        ops.rope_axes_cache_write(q, k, v, t.positions, s["pool"], t.slot_mapping, inv, SECTIONS, q_out=s["q"], layout="kv_first")
        ops.fog_decode(s["q"], s["pool"], s["table"], t.seq_lens, WIDTH * P, layout="kv_first", out=s["own"])
        ops.cross_attention(s["own"], ek, ev, t.query_start_loc, 1, ks, kl, max(STATES), out=s["out"])

    def inputs(s, i):
        s["have"].copy_(torch.tensor([[0, 16, 31], [15, 0, 100], [16, 47, 160], [WIDTH * P, 5, 32]][i]))
        s["count"].fill_(3)
        s["free"].copy_(torch.roll(free, 3 * i))
        s["qkv"].copy_(randn((b, HQ + 2 * HKV, D), torch.bfloat16, dev, 40 + i))
    eager, graph = fresh(), fresh()
    for s in (eager, graph):
        inputs(s, 0)
        step(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(graph)
    for i in (1, 2, 3, 0, 2):
        for s in (eager, graph):
            inputs(s, i)
        step(eager)
        g.replay()
        torch.cuda.synchronize()
        for name in ("pool", "table", "q", "own", "out"):
            assert torch.equal(eager[name], graph[name]), (i, name)
        for x, y in zip(eager["tables"], graph["tables"]):
            assert torch.equal(x, y)


def test_both_ways_into_the_cache(dev, monkeypatch):
    """rope_axes and the backend's own write with the fog on, or rope_axes_cache_write and fog_decode with the same bias:
    the same cache and the same rows."""
    from kessie_amd import kessie_attention as ka
    from kessie_amd import ops
    state = ka.KeSSieAttentionState()
    state.update(prompt_len=100, recall_positions={5, 30})
    monkeypatch.setattr(ka, "KESSIE_STATE", state)
    monkeypatch.setattr(ka, "_FOG_CACHE", ka._FogCache())
    inv, lens = inv_freq(D // 2, 10000.0, dev), [60, 17, 128]
    table = torch.arange(36, dtype=torch.int32, device=dev).view(3, WIDTH)
    free = torch.arange(36, 40, dtype=torch.int32, device=dev)
    qkv = randn((3, HQ + 2 * HKV, D), torch.bfloat16, dev, 5)
    pools = [randn((2, PAGES, P, HKV, D), torch.bfloat16, dev, 1) for _ in range(2)]
    meta = ka.KeSSieAttentionMetadata.build(table, lens, [1, 1, 1], P, free)
    assert meta.pages_taken == 1
    pos = three(meta.positions)
    q, k, v = qkv[:, :HQ].clone(), qkv[:, HQ:HQ + HKV].clone(), qkv[:, HQ + HKV:]
    ops.rope_axes(q, k, pos, inv, SECTIONS)
    one = ka.KeSSieAttentionImpl(HQ, D, D ** -0.5, HKV).forward(None, q.view(3, -1), k, v, pools[0], meta)
    q2, k2 = qkv[:, :HQ].clone(), qkv[:, HQ:HQ + HKV]
    ops.rope_axes_cache_write(q2, k2, v, pos, pools[1], meta.slot_mapping, inv, SECTIONS, layout="kv_first")
    bias = ka._FOG_CACHE.get_fog_bias_rows(meta.seq_lens, meta.max_seq_len, q.device, q.dtype, state.get())
    two = ops.fog_decode(q2, pools[1], meta.block_table, meta.seq_lens, meta.max_seq_len, fog_bias=bias, layout="kv_first")
    assert torch.equal(q, q2) and torch.equal(pools[0], pools[1]) and torch.equal(one.view(3, HQ, D), two)
