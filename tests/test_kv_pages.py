"""Pages of a KV cache that sequences share (include/ckb200_cache.h): tables, lengths, reference counts and page contents after every call, against the host's
walk over them one sequence after the other (q4_cache.Tables)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import q4_cache as host
from test_kv_cache_q4 import ALIGN, LIMIT, SHAPE, STATE, Device, gpu, handle, lib, near, up  # noqa: F401

BIG = 1 << 40
RESIZE = dict(page_table=256, table_stride=4, kv_lens=256, page_refs=256, new_lens=256, batch=2, num_pages=8, page_tokens=16, pages=256, planes=2, plane_stride=8 * 1280, page_bytes=1280,
              status=256, workspace=256, workspace_bytes=BIG, stream=None)
FORK = {**{n: RESIZE[n] for n in ("page_table", "table_stride", "kv_lens", "page_refs")}, "parent": 256, **{n: RESIZE[n] for n in ("batch", "num_pages", "page_tokens", "workspace",
                                                                                                                                "workspace_bytes", "stream")}}
COMPACT = {**{n: RESIZE[n] for n in ("page_table", "table_stride", "kv_lens", "page_refs", "batch", "num_pages", "page_tokens", "pages", "planes", "plane_stride", "page_bytes")},
           "live": 256, **{n: RESIZE[n] for n in ("workspace", "workspace_bytes", "stream")}}
COPY = dict(pages=256, planes=2, plane_stride=8 * 1280, page_bytes=1280, src=256, dst=256, count=2, num_pages=8, stream=None)
CALLS = {"ckb200_dev_kv_pages_resize": RESIZE, "ckb200_dev_kv_pages_fork": FORK, "ckb200_dev_kv_pages_compact": COMPACT, "ckb200_dev_kv_pages_copy": COPY}
CHANGES = [(dict(page_table=None), STATE), (dict(kv_lens=None), STATE), (dict(page_refs=None), STATE), (dict(new_lens=None), STATE), (dict(status=None), STATE), (dict(parent=None), STATE),
           (dict(src=None), STATE), (dict(dst=None), STATE), (dict(pages=None), STATE), (dict(workspace=None), STATE), (dict(workspace_bytes=16), STATE), (dict(workspace=264), ALIGN),
           (dict(page_refs=257), ALIGN), (dict(pages=264), ALIGN), (dict(live=257), ALIGN), (dict(parent=257), ALIGN), (dict(dst=257), ALIGN), (dict(new_lens=258), ALIGN),
           (dict(batch=-1), SHAPE), (dict(count=-1), SHAPE), (dict(table_stride=0), SHAPE), (dict(num_pages=0), SHAPE), (dict(page_tokens=0), SHAPE), (dict(planes=-1), SHAPE),
           (dict(page_bytes=1288), SHAPE), (dict(page_bytes=0), SHAPE), (dict(plane_stride=7 * 1280), SHAPE), (dict(plane_stride=8 * 1280 + 8), SHAPE), (dict(batch=4097), LIMIT),
           (dict(table_stride=1 << 27), LIMIT), (dict(table_stride=1 << 26, batch=32), LIMIT)]
REFUSED = [(name, change, code) for name, args in CALLS.items() for change, code in CHANGES if set(change) <= set(args)]


@pytest.mark.parametrize("name,change,code", REFUSED, ids=lambda v: v if isinstance(v, str) else (" ".join(v) if isinstance(v, dict) else ""))
def test_calls_that_are_refused(lib, name, change, code):  # noqa: F811
    lib.ckb200_clear_error()
    assert getattr(lib, name)(*{**CALLS[name], **change}.values()) == code
    assert lib.ckb200_last_error() == code
    lib.ckb200_clear_error()


def test_calls_without_sequences_do_nothing(lib):  # noqa: F811
    for name, args in CALLS.items():
        assert getattr(lib, name)(*{**args, **({"count": 0} if "count" in args else {"batch": 0})}.values()) == 0


def test_workspace_sizes(lib):  # noqa: F811
    assert lib.ckb200_kv_pages_workspace_bytes(0, 4, 8) == 0 and lib.ckb200_kv_pages_workspace_bytes(2, 0, 8) == 0
    assert lib.ckb200_kv_pages_workspace_bytes(4096, 1 << 20, 1 << 20) >= 4096 * (1 << 20) * 4


class Pages:
    """The same tables on the device."""

    def __init__(self, lib, model, page_bytes, planes, odd=0):  # noqa: F811
        self.lib, self.m, self.page_bytes, self.planes = lib, model, page_bytes, planes
        self.batch, self.stride = model.table.shape
        self.pages = len(model.refs)
        ints = up(np.concatenate([np.zeros(odd, dtype=np.int32), model.table.ravel(), model.lens, model.refs]))
        n = self.batch * self.stride
        self.table, self.lens, self.refs = ints[odd:odd + n].view(self.batch, self.stride), ints[odd + n:odd + n + self.batch], ints[odd + n + self.batch:]
        self.pool = up(model.pool)
        self.status, self.live = torch.full((self.batch,), 77, dtype=torch.int32, device="cuda"), torch.full((1,), 77, dtype=torch.int32, device="cuda")
        n = lib.ckb200_kv_pages_workspace_bytes(self.batch, self.stride, self.pages)
        self.ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")

    def tables(self):
        return self.table.data_ptr(), self.stride, self.lens.data_ptr(), self.refs.data_ptr()

    def whole(self):
        return self.pool.data_ptr() if self.planes else None, self.planes, self.pages * self.page_bytes, self.page_bytes

    def space(self, stream):
        return self.ws.data_ptr(), self.ws.numel(), handle(stream)

    def resize(self, new_lens, stream=None):
        self.asked = new_lens if isinstance(new_lens, torch.Tensor) else up(np.asarray(new_lens, dtype=np.int32))
        assert self.lib.ckb200_dev_kv_pages_resize(*self.tables(), self.asked.data_ptr(), self.batch, self.pages, self.m.pt, *self.whole(), self.status.data_ptr(), *self.space(stream)) == 0

    def fork(self, parent, stream=None):
        self.parent = parent if isinstance(parent, torch.Tensor) else up(np.asarray(parent, dtype=np.int32))
        assert self.lib.ckb200_dev_kv_pages_fork(*self.tables(), self.parent.data_ptr(), self.batch, self.pages, self.m.pt, *self.space(stream)) == 0

    def compact(self, stream=None):
        assert self.lib.ckb200_dev_kv_pages_compact(*self.tables(), self.batch, self.pages, self.m.pt, *self.whole(), self.live.data_ptr(), *self.space(stream)) == 0

    def same(self):
        torch.cuda.synchronize()
        for name, mine, want in (("table", self.table, self.m.table), ("lens", self.lens, self.m.lens), ("refs", self.refs, self.m.refs), ("pool", self.pool, self.m.pool)):
            assert np.array_equal(mine.cpu().numpy(), want), name
        assert (self.m.refs >= 0).all() and np.array_equal(np.bincount(self.m.table[self.m.table >= 0], minlength=self.pages), self.m.refs)


def make(lib, rng, batch, stride, pages, page_tokens, planes=3, page_bytes=160, odd=0):  # noqa: F811
    model = host.Tables(batch, stride, pages, page_tokens, rng.integers(0, 256, (planes, pages, page_bytes), dtype=np.uint8))
    return model, Pages(lib, model, page_bytes, planes, odd)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,stride,pages,page_tokens,planes,page_bytes", [(1, 1, 1, 16, 1, 16), (3, 4, 9, 16, 2, 320), (8, 6, 40, 16, 3, 5120), (33, 5, 90, 48, 1, 4112), (70, 9, 500, 16, 2, 160),
                                                                             (5, 300, 12, 16, 1, 32), (1100, 3, 2100, 16, 1, 16), (6, 5, 31, 64, 160, 2560), (4, 3, 12, 16, 0, 0),
                                                                             (310, 28, 9000, 16, 1, 16), (128, 64, 700, 16, 1, 16), (1700, 2, 1900, 16, 1, 16), (4096, 2, 4500, 16, 1, 16)])
def test_any_order_of_calls(gpu, batch, stride, pages, page_tokens, planes, page_bytes):  # noqa: F811
    """Grown, shrunk, freed, forked onto one another, compacted, with too little room now and then: after each call everything is what the host's walk gives."""
    rng = np.random.default_rng(batch * 7 + pages)
    m, d = make(gpu, rng, batch, stride, pages, page_tokens, planes, page_bytes, odd=batch % 3)
    refused = copied = 0
    for step in range(24):
        kind = step % 8
        if kind in (0, 1, 3, 5, 6):
            new = m.lens + rng.integers(-2 * page_tokens, 3 * page_tokens, batch) if kind != 5 else m.lens + 1
            new = np.where(rng.random(batch) < 0.1, [0, -1, stride * page_tokens + 1][step % 3], np.maximum(new, -1))
            before = m.refs.copy()
            want = m.resize(new)
            d.resize(new)
            d.same()
            assert np.array_equal(d.status.cpu().numpy(), want)
            refused, copied = refused + want.sum(), copied + (before > 1).sum()
        elif kind in (2, 4):
            parent = np.where(rng.random(batch) < 0.5, rng.integers(-1, batch + 1, batch), np.arange(batch))
            m.fork(parent)
            d.fork(parent)
            d.same()
        else:
            live = m.compact()
            d.compact()
            d.same()
            assert int(d.live) == live
    assert refused and (copied or batch == 1)


@pytest.mark.gpu
def test_branches_of_one_prompt(gpu):  # noqa: F811
    """Four continuations of a prompt: full pages shared, the last one copied for all but the last that names it; truncated and freed, everything is free again."""
    m, d = make(gpu, np.random.default_rng(0), 5, 8, 24, 16)
    for call, arg in (("resize", [40, 0, 0, 0, 0]), ("fork", [0, 0, 0, 0, -1]), ("resize", [41, 42, 43, 60, -1]), ("fork", [1, 0, 4, 2, 3]), ("resize", [33, 33, 33, 33, 80]), ("resize", [-1, 32, 16, 0, 0]),
                      ("resize", [50, 50, 50, 0, 0])):
        getattr(m, call)(arg)
        getattr(d, call)(arg)
        d.same()
        if call == "resize" and arg[0] == 41:
            assert sorted(m.refs[m.refs > 0].tolist()) == [1, 1, 1, 1, 1, 4, 4] and not int(d.status.sum())
    m.resize([0] * 5)
    d.resize([0] * 5)
    d.same()
    assert not m.refs.any()


@pytest.mark.gpu
def test_who_finds_no_room_stays(gpu):  # noqa: F811
    """Six pages, three sequences that share a partial page: the first copies it, the second needs more than is left and keeps sharing, so the third copies it too."""
    m, d = make(gpu, np.random.default_rng(1), 4, 8, 6, 16)
    for call, arg in (("resize", [20, 0, 0, 0]), ("fork", [0, 0, 0, 3]), ("resize", [30, 80, 21, 17])):
        want = getattr(m, call)(arg)
        getattr(d, call)(arg)
        d.same()
    assert want.tolist() == [0, 1, 0, 0] == d.status.cpu().tolist() and m.lens.tolist() == [30, 20, 21, 17]
    for arg, done in (([-1, -1, -1, 33], 1), ([-1, 0, -1, 33], 0)):
        assert m.resize(arg)[3] == done
        d.resize(arg)
        d.same()
        assert int(d.status[3]) == done


@pytest.mark.gpu
def test_many_pages(gpu):  # noqa: F811
    """A pool of 200000 pages and 4096 sequences, half of them freed and compacted away."""
    rng = np.random.default_rng(6)
    m, d = make(gpu, rng, 4096, 40, 200000, 16, planes=1, page_bytes=16)
    new = rng.integers(0, 640, 4096)
    for step in range(2):
        assert not m.resize(new).any()
        d.resize(new)
        d.same()
        new = np.where(rng.random(4096) < 0.5, 0, new)
    live = m.compact()
    d.compact()
    d.same()
    assert int(d.live) == live > 20000


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [8192, 8193])
@pytest.mark.parametrize("columns", [512, 513])
def test_thousands_at_once(gpu, pages, columns):  # noqa: F811
    """2048 pages and some more wanted by one call, forked, then as many moved by one compaction."""
    m, d = make(gpu, np.random.default_rng(7), 8, 1040, pages, 16, planes=1, page_bytes=16)
    for call, arg in (("resize", [16 * columns] * 4 + [0] * 4), ("resize", [-1] * 4 + [16 * columns] * 4), ("fork", [-1, -1, -1, -1, 5, -1, -1, 0]), ("resize", [0] * 4 + [16 * columns + 1] * 4)):
        getattr(m, call)(arg)
        getattr(d, call)(arg)
        d.same()
    live = m.compact()
    d.compact()
    d.same()
    assert int(d.live) == live


@pytest.mark.gpu
@pytest.mark.parametrize("page_bytes", [16, 1280, 4096, 4112, 40960])
def test_copies(gpu, page_bytes):  # noqa: F811
    """Pairs outside the pool, and of a page with itself, are passed over."""
    rng = np.random.default_rng(page_bytes)
    pool = rng.integers(0, 256, (5, 30, page_bytes), dtype=np.uint8)
    src, dst = np.array([3, 29, 3, -1, 30, 7, 8, 2 ** 31 - 1], dtype=np.int32), np.array([0, 1, 2, 4, 5, 7, 30, 6], dtype=np.int32)
    dev, s, t = up(pool), up(src), up(dst)
    assert gpu.ckb200_dev_kv_pages_copy(dev.data_ptr(), 5, 30 * page_bytes, page_bytes, s.data_ptr(), t.data_ptr(), len(src), 30, handle()) == 0
    torch.cuda.synchronize()
    pool[:, [0, 1, 2]] = pool[:, [3, 29, 3]]
    assert np.array_equal(dev.cpu().numpy(), pool)


@pytest.mark.gpu
def test_copies_beyond_32_bits(gpu):  # noqa: F811
    """Planes 5 GB apart."""
    page, pages = 1 << 20, 5000
    pool = torch.zeros(2, pages, page, dtype=torch.uint8, device="cuda")
    pool[1, 4999], pool[0, 4999] = 7, 5
    s, t = up(np.array([4999], dtype=np.int32)), up(np.array([4998], dtype=np.int32))
    assert gpu.ckb200_dev_kv_pages_copy(pool.data_ptr(), 2, pages * page, page, s.data_ptr(), t.data_ptr(), 1, pages, handle()) == 0
    torch.cuda.synchronize()
    assert (pool[1, 4998] == 7).all() and (pool[0, 4998] == 5).all() and not pool[:, :4998].any()


@pytest.mark.gpu
def test_tables_that_name_no_page(gpu):  # noqa: F811
    """Entries outside the pool among a sequence's columns are passed over by every call."""
    m, d = make(gpu, np.random.default_rng(2), 3, 4, 12, 16)
    m.resize([40, 20, 0])
    d.resize([40, 20, 0])
    m.refs[m.table[0, 1]] -= 1
    m.table[0, 1] = -1
    d.table[0, 1] = 12
    d.refs.copy_(up(m.refs))
    for call, arg in (("fork", [0, 1, 0]), ("resize", [41, 0, 17])):
        getattr(m, call)(arg)
        getattr(d, call)(arg)
    m.compact()
    d.compact()
    torch.cuda.synchronize()
    got = d.table.cpu().numpy()
    assert np.array_equal(np.where(got == 12, -1, got), m.table) and np.array_equal(d.refs.cpu().numpy(), m.refs) and np.array_equal(d.lens.cpu().numpy(), m.lens)


@pytest.mark.gpu
def test_a_captured_step(gpu):  # noqa: F811
    """One graph of a turn (fork, resize, compact), replayed with other parents and lengths."""
    rng = np.random.default_rng(9)
    m, d = make(gpu, rng, 6, 7, 60, 16)
    lens, parent = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.full((6,), -1, dtype=torch.int32, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        d.fork(parent, stream)
        d.resize(lens, stream)
        d.compact(stream)
    for step in range(6):
        p, n = rng.integers(-1, 6, 6).astype(np.int32), rng.integers(0, 100, 6).astype(np.int32)
        parent.copy_(up(p))
        lens.copy_(up(n))
        graph.replay()
        m.fork(p)
        want = m.resize(n)
        m.compact()
        d.same()
        assert np.array_equal(d.status.cpu().numpy(), want)


@pytest.mark.gpu
def test_a_conversation(gpu):  # noqa: F811
    """All of it as a server would use it: prompts stored, answered, branched, drafts taken back, sequences freed, the pool compacted - attention sees the rows that
    each sequence was given, whatever pages they lie in."""
    rng = np.random.default_rng(12)
    hkv, heads, hd, pt, pages, batch, stride = 2, 8, 128, 16, 60, 4, 12
    size = gpu.ckb200_kv_q4_page_bytes(hkv, pt, hd)
    model = host.Tables(batch, stride, pages, pt, np.zeros((2, pages, size), dtype=np.uint8))
    d = Pages(gpu, model, size, 2)
    told = [[np.zeros((0, hkv * hd), dtype=np.float32)] * 2 for _ in range(batch)]      # the K and V rows of each sequence

    def step(new_lens, tokens):
        d.resize(new_lens)
        model.resize(new_lens)
        x = rng.standard_normal((2, batch * tokens, hkv * hd)).astype(np.float32)
        q = rng.standard_normal((batch * tokens, heads * hd)).astype(np.float32)
        for b in range(batch):
            n = int(model.lens[b])
            t = min(tokens, n)
            for i in range(2):
                told[b][i] = np.concatenate([told[b][i][:n - t], x[i][b * tokens + tokens - t:(b + 1) * tokens]])
        kv = [up(a) for a in x]
        out, dq = torch.empty(batch * tokens, heads * hd, device="cuda"), up(q)
        where = (d.table.data_ptr(), stride, d.lens.data_ptr(), batch, tokens, pages, pt)
        pools = d.pool.data_ptr(), d.pool.data_ptr() + pages * size
        ws = torch.empty(max(16, gpu.ckb200_attention_q4cache_workspace_bytes(batch, tokens, heads, hkv, hd)), dtype=torch.uint8, device="cuda")
        assert gpu.ckb200_dev_kv_cache_store_q4(*pools, kv[0].data_ptr(), kv[1].data_ptr(), hkv * hd, hkv * hd, *where, hkv, hd, handle()) == 0
        assert gpu.ckb200_dev_attention_q4cache(dq.data_ptr(), heads * hd, *pools, out.data_ptr(), heads * hd, *where, heads, hkv, hd, 0, ws.data_ptr(), ws.numel(), handle()) == 0
        torch.cuda.synchronize()
        # the same rows in a cache of their own, page after page
        columns = -(-max(len(r[0]) for r in told) // pt)
        plain = host.Cache(hkv, hd, pt, batch * columns, np.arange(batch * columns).reshape(batch, columns), [len(r[0]) for r in told])
        for b, rows in enumerate(told):
            for pool, r in ((plain.k, rows[0]), (plain.v, rows[1])):
                for p in range(len(r)):
                    pool[b * columns + p // pt, :, p % pt] = host.quantize(r[p].reshape(hkv, hd))
        near(out.cpu().numpy(), *plain.attention(q, tokens, heads))
        assert np.array_equal(d.table.cpu().numpy(), model.table) and not d.status.any()

    step([40, 21, 0, 0], 40)                                    # prompts
    step([41, 22, 0, 0], 1)
    d.fork([0, 1, 0, 1])
    model.fork([0, 1, 0, 1])
    told[2], told[3] = list(told[0]), list(told[1])
    step([46, 27, 46, 27], 5)                                   # drafts on two branches of each
    for call in (d, model):
        call.resize([43, 24, 42, 22])                           # some are refused
    for b, n in enumerate([43, 24, 42, 22]):
        told[b] = [r[:n] for r in told[b]]
    step([44, 25, 43, 23], 1)
    for call in (d, model):
        call.resize([-1, 0, -1, -1])
        call.compact()
    told[1] = [r[:0] for r in told[1]]
    step([45, 1, 44, 24], 1)                                    # the freed one begins anew


@pytest.mark.gpu
@pytest.mark.parametrize("batch,stride,pages,page_tokens,free", [(3, 4, 30, 16, None), (40, 6, 200, 48, None), (1700, 3, 5000, 16, None), (4096, 2, 8192, 16, None), (4096, 2, 8193, 16, None),
                                                                 (700, 9, 9000, 16, None), (40, 180, 200, 48, 30), (60, 9000, 9000, 16, 40), (1700, 3, 1500, 16, None), (4096, 2, 3900, 16, None)])
def test_shared_pages_are_copied(gpu, batch, stride, pages, page_tokens, free):  # noqa: F811
    """A few prompts in all sequences, each continued: every one but the last that names a prompt's partial page gets a copy of it, counted here.  With little room (a small pool, or
    one sequence that holds all but `free` pages) some are refused and the others copied one by one."""
    rng = np.random.default_rng(batch + pages)
    prompts = max(1, batch // 50)
    m, d = make(gpu, rng, batch, stride, pages, page_tokens, planes=1, page_bytes=32)
    first = np.where(np.arange(batch) < prompts, rng.integers(1, page_tokens, batch) + page_tokens * rng.integers(0, min(stride, 4) - 1, batch), 0)
    parent = np.where(np.arange(batch) < prompts, -1, rng.integers(0, prompts, batch))
    if free:
        parent[-1] = -1
    for call, arg in (("resize", first), ("fork", parent)):
        getattr(m, call)(arg)
        getattr(d, call)(arg)
    new = np.full(batch, -1)
    if free:
        new[-1] = (int((m.refs == 0).sum()) - free) * page_tokens
        assert not m.resize(new)[-1]
        d.resize(new)
    d.same()
    before, lens = m.table.copy(), m.lens.copy()
    new = np.minimum(lens + 1 + page_tokens * (np.arange(batch) % 3 == 0), stride * page_tokens)
    want = m.resize(new)
    d.resize(new)
    d.same()
    assert np.array_equal(d.status.cpu().numpy(), want)
    last = np.maximum(lens - 1, 0) // page_tokens
    copies = int((m.table[np.arange(batch), last] != before[np.arange(batch), last]).sum())
    assert copies >= (20 if batch > 3 else 2) and want.any() == (free is not None or pages < batch)


@pytest.mark.gpu
def test_compacting_no_sequences_leaves_live_alone(gpu):  # noqa: F811
    m, d = make(gpu, np.random.default_rng(3), 2, 3, 9, 16)
    for call in (m, d):
        call.resize([20, 40])
        call.resize([0, 40])
    assert gpu.ckb200_dev_kv_pages_compact(*d.tables(), 0, d.pages, m.pt, *d.whole(), d.live.data_ptr(), *d.space(None)) == 0
    d.same()
    assert int(d.live) == 77
