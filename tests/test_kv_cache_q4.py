"""Rows of a paged 4-bit KV cache and the attention over them (include/ckb200_cache.h) against the host's: q4_cache.py."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

import q4_cache as host
from q4_cache import BLOCK, Cache

SHAPE, ALIGN, NO_DEVICE, LIMIT, STATE = 2, 3, 4, 6, 7


@pytest.fixture(scope="module")
def lib(pkg):
    """The library with argument types, not initialised: refusals need no device."""
    lib = pkg.load_lib()
    pkg.cache_api.bind_cache_api(lib)
    return lib


@pytest.fixture
def gpu(ck, lib):
    return lib


# ------------------------------------------------------------------ refusals, and where rows lie: no device

STORE = dict(k_pages=256, v_pages=256, k=256, v=256, k_stride=256, v_stride=256, page_table=256, table_stride=4, kv_lens=256, batch=2, num_tokens=1, num_pages=8, page_tokens=16,
             num_kv_heads=2, head_dim=128, stream=None)
LOAD = {n: STORE[n] for n in ("k", "v", "k_stride", "v_stride", "k_pages", "v_pages", "page_table", "table_stride", "kv_lens", "batch", "num_tokens", "num_pages", "page_tokens",
                              "num_kv_heads", "head_dim", "stream")}
ATTEND = dict(q=256, q_stride=512, k_pages=256, v_pages=256, out=256, out_stride=512, page_table=256, table_stride=4, kv_lens=256, batch=2, num_tokens=1, num_pages=8, page_tokens=16,
              num_heads=4, num_kv_heads=2, head_dim=128, sliding_window=0, workspace=256, workspace_bytes=1 << 40, stream=None)
ROPE = dict(q=256, k=256, v=256, k_pages=256, v_pages=256, cos_cache=256, sin_cache=256, rope_positions=100, page_table=256, table_stride=4, kv_lens=256, batch=2, num_pages=8, page_tokens=16,
            num_heads=4, num_kv_heads=2, head_dim=128, stream=None)
CALLS = {"ckb200_dev_rope_kv_store_q4": ROPE, "ckb200_dev_kv_cache_store_q4": STORE, "ckb200_dev_kv_cache_load_q4": LOAD, "ckb200_dev_attention_q4cache": ATTEND}
COMMON = [(dict(k_pages=None), STATE), (dict(v_pages=None), STATE), (dict(page_table=None), STATE), (dict(kv_lens=None), STATE), (dict(batch=-1), SHAPE), (dict(num_tokens=-1), SHAPE),
          (dict(num_pages=0), SHAPE), (dict(table_stride=0), SHAPE), (dict(page_tokens=0), SHAPE), (dict(page_tokens=24), SHAPE), (dict(num_kv_heads=0), SHAPE), (dict(head_dim=80), SHAPE),
          (dict(head_dim=32), SHAPE), (dict(k_pages=264), ALIGN), (dict(v_pages=257), ALIGN), (dict(kv_lens=258), ALIGN), (dict(table_stride=1 << 27), LIMIT), (dict(num_kv_heads=1025), LIMIT)]
ROWS = [(dict(k=None), STATE), (dict(v=None), STATE), (dict(k=257), ALIGN), (dict(k_stride=255), SHAPE), (dict(v_stride=-256), SHAPE), (dict(batch=1 << 30, num_tokens=1 << 30), LIMIT)]
OWN = [(dict(q=None), STATE), (dict(out=None), STATE), (dict(q=258), ALIGN), (dict(num_heads=0), SHAPE), (dict(num_heads=5), SHAPE), (dict(sliding_window=-1), SHAPE), (dict(q_stride=511), SHAPE),
       (dict(out_stride=0), SHAPE), (dict(batch=1 << 20, num_tokens=1 << 20), LIMIT), (dict(batch=1 << 15, num_tokens=1 << 15), LIMIT), (dict(workspace=None), STATE),
       (dict(workspace_bytes=1000), STATE), (dict(workspace=264), ALIGN)]
TURN = [(dict(q=None), STATE), (dict(k=None), STATE), (dict(cos_cache=None), STATE), (dict(sin_cache=257), ALIGN), (dict(v=258), ALIGN), (dict(rope_positions=0), SHAPE), (dict(num_heads=0), SHAPE),
        (dict(batch=1 << 28), LIMIT)]
REFUSED = [(name, change, code) for name, args in CALLS.items() for change, code in COMMON + (OWN if "attention" in name else (TURN if "rope" in name else ROWS)) if set(change) <= set(args)]


@pytest.mark.parametrize("name,change,code", REFUSED, ids=lambda v: v if isinstance(v, str) else (" ".join(v) if isinstance(v, dict) else ""))
def test_calls_that_are_refused(lib, name, change, code):
    lib.ckb200_clear_error()
    assert getattr(lib, name)(*{**CALLS[name], **change}.values()) == code
    assert lib.ckb200_last_error() == code
    lib.ckb200_clear_error()


@pytest.mark.parametrize("name", CALLS)
def test_calls_without_rows_do_nothing(lib, name):
    for change in (dict(batch=0), dict(num_tokens=0)):
        if set(change) <= set(CALLS[name]):
            assert getattr(lib, name)(*{**CALLS[name], **change}.values()) == 0


def test_where_rows_lie(lib):
    table = np.array([3, 0, -1, 8, 2 ** 31 - 1, -2 ** 31, 7], dtype=np.int32)
    at = lambda pos, pages=8, heads=3, hd=96, head=1, pt=16: lib.ckb200_kv_q4_row_offset(table.ctypes.data, len(table), pages, pt, heads, hd, head, pos)      # noqa: E731
    row = 96 // 32 * BLOCK
    assert lib.ckb200_kv_q4_page_bytes(3, 16, 96) == 3 * 16 * row
    assert at(0) == ((3 * 3 + 1) * 16 + 0) * row and at(17) == ((0 * 3 + 1) * 16 + 1) * row and at(6 * 16 + 15) == ((7 * 3 + 1) * 16 + 15) * row
    # no entry, an entry beyond the pool, positions before the first and behind the last column
    assert [at(p) for p in (32, 47, 48, 64, 80, -1, -2 ** 31, 7 * 16, 2 ** 31 - 1)] == [-1] * 9
    assert at(96, pages=7) == -1 and at(0, head=3) == -1 and at(0, head=-1) == -1 and at(0, hd=80) == -1 and at(0, pt=8) == -1
    far = np.array([2 ** 20], dtype=np.int32)
    assert lib.ckb200_kv_q4_row_offset(far.ctypes.data, 1, 2 ** 21, 64, 8, 128, 7, 63) == ((2 ** 20 * 8 + 7) * 64 + 63) * 80 > 2 ** 32


# ------------------------------------------------------------------ on the device

def up(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def handle(stream=None):
    return (stream or torch.cuda.current_stream()).cuda_stream or 1


def scattered(rng, lens, page_tokens, spare=2, extra_columns=1, hole=False):
    """A table whose sequences lie in pages of a random order, as many columns as the longest needs and more; (table, pages).  hole: one column of the longest
    sequence has no page, another names one that does not exist."""
    used = [-(-max(0, n) // page_tokens) for n in lens]
    pages = sum(used) + spare
    order = rng.permutation(pages)
    table = np.full((len(lens), max(used + [1]) + extra_columns), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    if hole:
        b = int(np.argmax(lens))
        table[b, used[b] // 2] = -1
        table[b, 0] = pages
    return table, pages


class Device:
    """A host cache's copy on the device, and the calls on it."""

    def __init__(self, lib, cache):
        self.lib, self.c = lib, cache
        self.k, self.v, self.table, self.lens = up(cache.k), up(cache.v), up(cache.table), up(cache.lens)

    def where(self, tokens):
        c = self.c
        return (self.table.data_ptr(), c.table.shape[1], self.lens.data_ptr(), len(c.lens), tokens, c.pages, c.page_tokens)

    def store(self, k, v, tokens, stream=None):
        assert self.lib.ckb200_dev_kv_cache_store_q4(self.k.data_ptr(), self.v.data_ptr(), k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), *self.where(tokens), self.c.kv_heads,
                                                     self.c.head_dim, handle(stream)) == 0

    def load(self, k, v, tokens, stream=None):
        assert self.lib.ckb200_dev_kv_cache_load_q4(k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), self.k.data_ptr(), self.v.data_ptr(), *self.where(tokens), self.c.kv_heads,
                                                    self.c.head_dim, handle(stream)) == 0

    def workspace(self, tokens, heads):
        n = self.lib.ckb200_attention_q4cache_workspace_bytes(len(self.c.lens), tokens, heads, self.c.kv_heads, self.c.head_dim)
        return torch.full((max(16, n),), 255, dtype=torch.uint8, device="cuda")

    def attend(self, q, out, tokens, heads, window, workspace, stream=None):
        assert self.lib.ckb200_dev_attention_q4cache(q.data_ptr(), q.stride(0), self.k.data_ptr(), self.v.data_ptr(), out.data_ptr(), out.stride(0), *self.where(tokens), heads,
                                                     self.c.kv_heads, self.c.head_dim, window, workspace.data_ptr(), workspace.numel(), handle(stream)) == 0

    def attention(self, q, tokens, heads, window=0):
        out = torch.full((len(q), heads * self.c.head_dim), 9.0, device="cuda")
        self.attend(up(q), out, tokens, heads, window, self.workspace(tokens, heads))
        torch.cuda.synchronize()
        return out.cpu().numpy()


def random_cache(rng, kv_heads, head_dim, page_tokens, lens, fill=True, **kw):
    table, pages = scattered(rng, lens, page_tokens, **kw)
    c = Cache(kv_heads, head_dim, page_tokens, pages, table, lens)
    if fill:                                                    # pages that nobody holds, and rows behind the last token, stay NaN
        for b, n in enumerate(lens):
            for i in range(-(-max(0, n) // page_tokens)):
                page, rows = table[b, i], min(page_tokens, n - i * page_tokens)
                if 0 <= page < pages:
                    for pool in (c.k, c.v):
                        x = rng.standard_normal((kv_heads, rows, head_dim)).astype(np.float32)
                        x[..., ::19] *= 3
                        pool[page, :, :rows] = host.quantize(x)
    return c


def edge_rows(rng, n, width):
    """Rows whose blocks hold what a quantiser can trip over."""
    x = rng.standard_normal((n, width)).astype(np.float32)
    flat = x.reshape(-1, 32)
    kinds = [np.zeros(32), np.full(32, -7.25), np.full(32, 65504.0), np.full(32, -65504.0), np.full(32, 65520.0), np.linspace(-65504, 65504, 32), np.full(32, 1e-9),
             np.linspace(0, 1e-7, 32), np.linspace(-3e38, 3e38, 32), np.arange(32) * 0.5, -np.arange(32) / 3]
    for i in range(0, len(flat), 3):
        kind = kinds[(i // 3) % (len(kinds) + 4)] if (i // 3) % (len(kinds) + 4) < len(kinds) else None
        if kind is not None:
            flat[i] = kind
        else:
            flat[i, i % 32] = [np.nan, np.inf, -np.inf, -0.0][(i // 3) % (len(kinds) + 4) - len(kinds)]
    return x


ROW_CASES = [
    # kv_heads, head_dim, page_tokens, lens, tokens, hole
    (1, 64, 16, [1], 1, False), (2, 64, 16, [5, 16, 17, 0], 1, False), (3, 96, 48, [100, 3, 47], 7, False), (8, 128, 64, [130, 64, 1], 33, False),
    (2, 192, 16, [40, 9], 40, False), (1, 256, 32, [33], 50, False), (2, 128, 16, [70, 20], 70, True), (5, 64, 128, [-4, 1000], 3, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,head_dim,page_tokens,lens,tokens,hole", ROW_CASES)
@pytest.mark.parametrize("shift", [0, 1], ids=["aligned", "odd"])
def test_rows_stored_and_read_back(gpu, kv_heads, head_dim, page_tokens, lens, tokens, hole, shift):
    """Every byte of the pools, and the fp32 rows that come back, are those of the host's fp32 steps: rows at odd addresses and distances, blocks that no code can hold,
    sequences shorter than the call, entries without a page, and 1000 tokens by kv_lens where the table has fewer."""
    rng = np.random.default_rng(kv_heads * 1000 + head_dim + tokens)
    c = random_cache(rng, kv_heads, head_dim, page_tokens, [min(n, 200) for n in lens], hole=hole)
    c.lens[:] = lens
    dev = Device(gpu, c)
    n, rows = kv_heads * head_dim, len(lens) * tokens
    x = [edge_rows(rng, rows, n) for _ in range(2)]
    wide = torch.full((rows, 2 * n + 5), 3.0, device="cuda")
    k, v = wide[:, shift:shift + n], wide[:, n + 2 * shift:2 * n + 2 * shift]
    k.copy_(up(x[0]))
    v.copy_(up(x[1]))
    dev.store(k, v, tokens)
    c.store(x[0], x[1], tokens)
    back = torch.full((rows, 2 * n + 5), 7.0, device="cuda")
    dev.load(back[:, shift:shift + n], back[:, n + 2 * shift:2 * n + 2 * shift], tokens)
    torch.cuda.synchronize()
    for mine, want in ((dev.k, c.k), (dev.v, c.v)):
        got = mine.cpu().numpy().reshape(want.shape)
        # the sign of a minimum that is zero may be either
        a, b = (p.reshape(-1, BLOCK).copy() for p in (got, want))
        for p in (a, b):
            zero = (p[:, 2] == 0) & (p[:, 3] == 128)
            p[zero, 3] = 0
        assert np.array_equal(a, b)
    got = back.cpu().numpy()
    used = np.zeros(2 * n + 5, dtype=bool)
    for i, pool in enumerate((c.k, c.v)):
        lo = shift if i == 0 else n + 2 * shift
        used[lo:lo + n] = True
        for b in range(len(lens)):
            for t in range(tokens):
                at = c.place(b, c.length(b) - tokens + t)
                want = host.values(pool[at[0], :, at[1]], np.float32).reshape(-1) if at else np.zeros(n, dtype=np.float32)
                assert np.array_equal(got[b * tokens + t, lo:lo + n], want, equal_nan=True)
    assert (got[:, ~used] == 7.0).all()


@pytest.mark.gpu
def test_rows_are_those_of_the_row_dequantiser(gpu):
    """A cache row is a row of block_q4_1: the library's own dequantiser reads it."""
    rng = np.random.default_rng(5)
    c = random_cache(rng, 2, 128, 16, [16], spare=0, extra_columns=0)
    dev = Device(gpu, c)
    gpu.ckb200_dev_dequant_q4_1_row.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
    y = torch.empty(2 * 16 * 128, device="cuda")
    assert gpu.ckb200_dev_dequant_q4_1_row(dev.k.data_ptr(), y.data_ptr(), y.numel(), handle()) == 0
    torch.cuda.synchronize()
    assert np.array_equal(y.cpu().numpy().reshape(2, 16, 128), host.values(c.k[0], np.float32))


def near(got, want, off):
    bad = ~(np.abs(got - want) <= off)
    assert not bad.any(), f"{bad.sum()} of {bad.size}, the worst {np.abs(got - want).max():.3g} where {off[np.unravel_index(np.nanargmax(np.abs(got - want) - off), off.shape)]:.3g} is allowed"
    # errors of single roundings do not add up to the worst case: together they stay within the square root of their number
    if np.linalg.norm(want):
        assert np.linalg.norm(got - want) <= 2e-5 * np.linalg.norm(want)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,head_dim,page_tokens,lens", [(1, 1, 64, 16, [1]), (14, 2, 64, 16, [5, 0, 48, 49]), (5, 5, 96, 48, [100]), (32, 8, 128, 64, [64, 65, 3]), (3, 1, 192, 16, [20, 31]),
                                                                      (6, 3, 256, 32, [33, 150, -1])])
def test_a_turn_rotates_and_stores(gpu, heads, kv_heads, head_dim, page_tokens, lens):
    """q and the pools after one call are, bit for bit, those of the rotation in fp32 and of the host's store; the last sequence's position is behind the tables and
    it stays as it is, as does one of length 0."""
    rng = np.random.default_rng(heads + head_dim)
    c = random_cache(rng, kv_heads, head_dim, page_tokens, lens)
    dev, batch, half = Device(gpu, c), len(lens), head_dim // 2
    positions = max(lens) if batch > 1 and lens[-1] == max(lens) else max(lens) + 2
    positions = lens[-1] - 1 if batch > 2 and lens[-1] == max(lens) else positions
    angle = np.arange(positions)[:, None] * (10000.0 ** (-np.arange(half) / half))[None]
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    q, k, v = (rng.standard_normal((batch, n, head_dim)).astype(np.float32) for n in (heads, kv_heads, kv_heads))

    def turned(x):
        y = x.copy()
        for b, n in enumerate(lens):
            if 0 < n <= positions:
                u, w, co, si = x[b, :, :half], x[b, :, half:], cos[n - 1], sin[n - 1]
                y[b, :, :half], y[b, :, half:] = u * co - w * si, u * si + w * co
        return y

    d = [up(a) for a in (q, k, v, cos, sin)]
    assert gpu.ckb200_dev_rope_kv_store_q4(d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), dev.k.data_ptr(), dev.v.data_ptr(), d[3].data_ptr(), d[4].data_ptr(), positions,
                                           dev.table.data_ptr(), c.table.shape[1], dev.lens.data_ptr(), batch, c.pages, page_tokens, heads, kv_heads, head_dim, handle()) == 0
    torch.cuda.synchronize()
    assert np.array_equal(d[0].cpu().numpy(), turned(q)) and np.array_equal(d[1].cpu().numpy(), k)
    c.lens = np.where(c.lens > positions, 0, c.lens).astype(np.int32)
    c.store(turned(k).reshape(batch, -1), v.reshape(batch, -1), 1)
    assert np.array_equal(dev.k.cpu().numpy().reshape(c.k.shape), c.k) and np.array_equal(dev.v.cpu().numpy().reshape(c.v.shape), c.v)


ATTENTION_CASES = [
    # heads, kv_heads, head_dim, page_tokens, lens, tokens, window
    (1, 1, 64, 16, [1], 1, 0), (4, 4, 64, 16, [0, 1, 15, 16, 17, 31, 32, 33], 1, 0), (14, 2, 64, 16, [77], 1, 0), (7, 1, 96, 48, [47, 48, 49, 200], 1, 0),
    (8, 1, 128, 64, [300, 64, 65], 1, 0), (32, 8, 128, 64, [513], 1, 0), (9, 1, 128, 32, [127, 128, 129], 1, 0), (24, 2, 64, 16, [250, 3], 1, 0), (2, 1, 192, 16, [90, 31], 1, 0),
    (10, 2, 256, 16, [100, 255, 1], 1, 0), (40, 1, 64, 16, [150], 1, 0), (4, 2, 128, 16, [400, 90, 20], 1, 33), (4, 2, 64, 128, [1000], 1, 1), (3, 1, 64, 16, [66], 1, 1000),
    (8, 2, 128, 64, [130, 5, 0, 64], 5, 0), (12, 4, 64, 16, [40, 39, 7, 8], 8, 0), (4, 4, 96, 16, [64], 64, 0), (8, 1, 128, 32, [200, 30], 33, 0), (6, 2, 256, 16, [70], 9, 0), (5, 5, 192, 32, [80], 21, 17),
    # more parts of one sequence than a warp has lanes, sequences by the dozen, more of them than threads in a block
    (3, 1, 64, 16, [9000], 1, 0), (2, 1, 128, 32, [5000, 17], 2, 0), (4, 2, 64, 16, [(37 * i) % 411 for i in range(90)], 1, 0), (1, 1, 64, 16, [i % 19 for i in range(700)], 1, 0),
    (5, 1, 256, 16, [4500], 1, 2 ** 31 - 1),
    # the same with several blocks of query rows and kv heads, and a stretch in a dozen parts
    (16, 4, 64, 16, [(29 * i) % 61 for i in range(150)], 9, 20), (3, 3, 96, 16, [(31 * i) % 50 for i in range(200)], 3, 0), (24, 24, 64, 16, [2400], 1, 0), (24, 12, 128, 32, [1300, 5, 1299], 4, 0),
    # tables with room for so much that four CTAs an SM are taken
    (40, 8, 128, 16, [2100] + [(13 * i) % 90 for i in range(40)], 1, 0), (16, 8, 128, 64, [9, 4200, 0] + [(17 * i) % 70 for i in range(25)], 3, 700),
    (16, 2, 64, 16, [300, 90], 17, 40), (2, 2, 128, 16, [130], 130, 16), (4, 1, 128, 16, [3000, 5, 2049], 1, 0), (8, 8, 64, 256, [2500], 3, 2048), (4, 1, 128, 64, [50], 100, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,head_dim,page_tokens,lens,tokens,window", ATTENTION_CASES)
def test_attention(gpu, heads, kv_heads, head_dim, page_tokens, lens, tokens, window):
    rng = np.random.default_rng(heads * 100 + head_dim + len(lens) + tokens)
    c = random_cache(rng, kv_heads, head_dim, page_tokens, lens)
    q = rng.standard_normal((len(lens) * tokens, heads * head_dim)).astype(np.float32)
    got = Device(gpu, c).attention(q, tokens, heads, window)
    near(got, *c.attention(q, tokens, heads, window))
    for b, n in enumerate(lens):                                # rows before the first token see nothing
        assert (got[b * tokens:b * tokens + max(0, tokens - n)] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [1e-3, 30.0], ids=["small", "large"])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_attention_of_other_magnitudes(gpu, head_dim, spread):
    """Values, keys and queries three orders of magnitude apart, and blocks of one sequence whose steps differ by 2^12."""
    rng = np.random.default_rng(head_dim)
    c = random_cache(rng, 2, head_dim, 16, [200, 45])
    for b, n in enumerate(c.lens):
        for i in range(-(-int(n) // 16)):
            page, rows = c.table[b, i], min(16, int(n) - 16 * i)
            x = rng.standard_normal((2, rows, head_dim)).astype(np.float32) * np.float32(spread) * (np.float32(2.0) ** rng.integers(-6, 7, (2, rows, 1)).astype(np.float32))
            c.v[page, :, :rows] = host.quantize(x)
            c.k[page, :, :rows] = host.quantize(rng.standard_normal((2, rows, head_dim)).astype(np.float32) / np.float32(spread))
    q = (rng.standard_normal((2, 8 * head_dim)) * spread).astype(np.float32)
    near(Device(gpu, c).attention(q, 1, 8), *c.attention(q, 1, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 6])
def test_tokens_without_a_page_are_not_seen(gpu, tokens):
    rng = np.random.default_rng(3)
    c = random_cache(rng, 2, 64, 16, [100, 50], hole=True)
    q = rng.standard_normal((2 * tokens, 4 * 64)).astype(np.float32)
    near(Device(gpu, c).attention(q, tokens, 4), *c.attention(q, tokens, 4))
    c.table[0] = -1
    dev = Device(gpu, c)
    got = dev.attention(q, tokens, 4)
    assert (got[:tokens] == 0).all()
    near(got, *c.attention(q, tokens, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_rows_that_are_no_numbers(gpu, which, head_dim):
    """The third of five new tokens has a block of NaN: the tokens before it, and all with a window that has passed it, are as without it; those that see it have NaN
    in that block's channels (in all for a key)."""
    rng = np.random.default_rng(11)
    c = random_cache(rng, 1, head_dim, 16, [90])
    page, slot = c.place(0, 87)
    pool = c.k if which == "k" else c.v
    pool[page, 0, slot, BLOCK:BLOCK + 4] = 255
    q = rng.standard_normal((5, 4 * head_dim)).astype(np.float32)
    for window, hit in ((0, [2, 3, 4]), (2, [2, 3])):
        got = Device(gpu, c).attention(q, 5, 4, window)
        want, off = c.attention(q, 5, 4, window)
        spoilt = np.isnan(want)
        assert sorted(set(np.flatnonzero(spoilt.any(1)))) == hit and np.array_equal(np.isnan(got), spoilt)
        near(np.where(spoilt, 0, got), np.where(spoilt, 0, want), np.where(spoilt, 0, off))


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim", [64, 128])
def test_a_row_that_is_no_number_spoils_its_block_alone(gpu, head_dim):
    """A value block of NaN early in a long context, seen by every query: the other blocks' channels are as exact as without it."""
    rng = np.random.default_rng(13)
    c = random_cache(rng, 1, head_dim, 16, [400])
    page, slot = c.place(0, 10)
    c.v[page, 0, slot, :4] = 255
    q = rng.standard_normal((1, 4 * head_dim)).astype(np.float32)
    got = Device(gpu, c).attention(q, 1, 4).reshape(4, head_dim)
    want, off = (a.reshape(4, head_dim) for a in c.attention(q, 1, 4))
    assert np.isnan(got[:, :32]).all() and np.isnan(want[:, :32]).all()
    near(got[:, 32:], want[:, 32:], off[:, 32:])


@pytest.mark.gpu
def test_attention_rows_of_wider_tensors(gpu):
    """q is a part of a fused projection's rows at an odd place, out a part of a wider tensor whose other columns stay as they are."""
    rng = np.random.default_rng(8)
    c = random_cache(rng, 2, 128, 32, [77, 130])
    q = rng.standard_normal((6, 4 * 128)).astype(np.float32)
    wide_q, wide_out = torch.full((6, 1001), float("nan"), device="cuda"), torch.full((6, 601), 5.0, device="cuda")
    wide_q[:, 333:845] = up(q)
    dev = Device(gpu, c)
    dev.attend(wide_q[:, 333:845], wide_out[:, 7:519], 3, 4, 0, dev.workspace(3, 4))
    torch.cuda.synchronize()
    near(wide_out[:, 7:519].cpu().numpy(), *c.attention(q, 3, 4))
    assert (wide_out[:, :7] == 5).all() and (wide_out[:, 519:] == 5).all()


@pytest.mark.gpu
def test_pool_beyond_32_bits(gpu):
    """Pages whose bytes begin past 2^32, and rows that end in the pool's last byte."""
    pages, hkv, hd, pt = 55000, 8, 128, 128
    size = gpu.ckb200_kv_q4_page_bytes(hkv, pt, hd)
    assert size * (pages - 3) > 2 ** 32
    lens = np.array([200, 256], dtype=np.int32)
    table = np.array([[pages - 3, 1], [pages - 2, pages - 1]], dtype=np.int32)
    small = Cache(hkv, hd, pt, 4, [[0, 1], [2, 3]], lens)
    rng = np.random.default_rng(4)
    x = [rng.standard_normal((512, hkv * hd)).astype(np.float32) for _ in range(2)]
    small.store(x[0], x[1], 256)
    pools = [torch.empty(pages * size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    t, ln, k, v = up(table), up(lens), up(x[0]), up(x[1])
    where = (t.data_ptr(), 2, ln.data_ptr(), 2, 256, pages, pt, hkv, hd)
    assert gpu.ckb200_dev_kv_cache_store_q4(pools[0].data_ptr(), pools[1].data_ptr(), k.data_ptr(), v.data_ptr(), hkv * hd, hkv * hd, *where, handle()) == 0
    back = torch.empty(2, 512, hkv * hd, device="cuda")
    assert gpu.ckb200_dev_kv_cache_load_q4(back[0].data_ptr(), back[1].data_ptr(), hkv * hd, hkv * hd, pools[0].data_ptr(), pools[1].data_ptr(), *where, handle()) == 0
    q = rng.standard_normal((2, hkv * hd)).astype(np.float32)
    out, dq = torch.empty(2, hkv * hd, device="cuda"), up(q)
    ws = torch.empty(max(16, gpu.ckb200_attention_q4cache_workspace_bytes(2, 1, hkv, hkv, hd)), dtype=torch.uint8, device="cuda")
    assert gpu.ckb200_dev_attention_q4cache(dq.data_ptr(), hkv * hd, pools[0].data_ptr(), pools[1].data_ptr(), out.data_ptr(), hkv * hd, t.data_ptr(), 2, ln.data_ptr(), 2, 1, pages, pt,
                                            hkv, hkv, hd, 0, ws.data_ptr(), ws.numel(), handle()) == 0
    torch.cuda.synchronize()
    assert torch.equal(pools[0][(pages - 2) * size:(pages - 1) * size].cpu(), torch.from_numpy(small.k[2].reshape(-1)))
    for i, pool in enumerate((small.k, small.v)):
        want = host.values(pool[small.table[1]].transpose(1, 0, 2, 3).reshape(hkv, 256, -1), np.float32).transpose(1, 0, 2).reshape(256, -1)
        assert np.array_equal(back[i, 256:].cpu().numpy(), want)
    near(out.cpu().numpy(), *small.attention(q, 1, hkv))


@pytest.mark.gpu
def test_sequences_of_millions_of_tokens(gpu):
    """2^24 tokens whose table names one page over and over (and 16 more in a second sequence): the result is that of the page's tokens, whatever the number of units,
    which passes 2^20 here, and of the partial results that are joined."""
    rng = np.random.default_rng(17)
    hkv, hd, columns = 8, 64, 1 << 20
    small = random_cache(rng, hkv, hd, 16, [16, 16], spare=0)
    dev = Device(gpu, small)
    table = np.full((2, columns), small.table[0, 0], dtype=np.int32)
    table[1, 0] = small.table[1, 0]
    big, lens = up(table), up(np.array([columns * 16, 16], dtype=np.int32))
    q = rng.standard_normal((2, 16 * hd)).astype(np.float32)
    dq, out = up(q), torch.zeros(2, 16 * hd, device="cuda")
    ws = dev.workspace(1, 16)
    assert gpu.ckb200_dev_attention_q4cache(dq.data_ptr(), 16 * hd, dev.k.data_ptr(), dev.v.data_ptr(), out.data_ptr(), 16 * hd, big.data_ptr(), columns, lens.data_ptr(), 2, 1, 2, 16, 16, hkv,
                                            hd, 0, ws.data_ptr(), ws.numel(), handle()) == 0
    torch.cuda.synchronize()
    want, off = small.attention(q, 1, 16)
    # 2^24 weights are added by 444 CTAs in chunks of 32: 2^10 roundings in a row at the most, where the bound has 16
    near(out.cpu().numpy(), want, off + 2.0 ** -13)


@pytest.mark.gpu
def test_two_calls_at_once_and_graphs(gpu):
    """Two streams with workspaces of their own, at once; and a step (store, attention) that is captured once and replayed while its sequences grow, its graph and another's
    sharing one workspace in turn."""
    rng = np.random.default_rng(21)
    caches = [random_cache(rng, 2, 128, 32, [700, 40]), random_cache(rng, 2, 128, 32, [33, 900])]
    devs = [Device(gpu, c) for c in caches]
    qs = [rng.standard_normal((2, 8 * 128)).astype(np.float32) for _ in caches]
    dq, outs = [up(q) for q in qs], [torch.zeros(2, 8 * 128, device="cuda") for _ in qs]
    spaces, streams = [d.workspace(1, 8) for d in devs], [torch.cuda.Stream() for _ in devs]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, d in enumerate(devs):
            d.attend(dq[i], outs[i], 1, 8, 0, spaces[i], streams[i])
    torch.cuda.synchronize()
    for i, c in enumerate(caches):
        near(outs[i].cpu().numpy(), *c.attention(qs[i], 1, 8))

    rows = [torch.zeros(2, 4, 2 * 128, device="cuda") for _ in caches]
    graphs = []
    for i, d in enumerate(devs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            d.store(rows[i][0], rows[i][1], 2, streams[i])
            d.attend(dq[i], outs[i], 1, 8, 0, spaces[0], streams[i])
        graphs.append(g)
    for step in range(3):
        for i, c in enumerate(caches):
            c.lens += [1, 2][step % 2]
            x = rng.standard_normal((2, 4, 2 * 128)).astype(np.float32)
            qs[i] = rng.standard_normal((2, 8 * 128)).astype(np.float32)
            devs[i].lens.copy_(up(c.lens))
            rows[i].copy_(up(x))
            dq[i].copy_(up(qs[i]))
            graphs[i].replay()
            c.store(x[0], x[1], 2)
        torch.cuda.synchronize()
        for i, c in enumerate(caches):
            near(outs[i].cpu().numpy(), *c.attention(qs[i], 1, 8))


@pytest.mark.gpu
def test_results_do_not_change_from_run_to_run(gpu):
    rng = np.random.default_rng(2)
    c = random_cache(rng, 4, 128, 64, [1500, 3, 800])
    q = rng.standard_normal((3, 16 * 128)).astype(np.float32)
    dev = Device(gpu, c)
    first = dev.attention(q, 1, 16)
    assert all(np.array_equal(first, dev.attention(q, 1, 16)) for _ in range(5))


def within(got, want, off):
    """Blocks that the store holds to be beyond fp16 read as NaN, in the channels that they are in; everything else is within its bound."""
    spoilt = np.isnan(want)
    assert np.array_equal(np.isnan(got), spoilt)
    far = np.where(spoilt, 0, np.abs(got - want) / np.where(spoilt, 1, np.maximum(off, 1e-300)))
    assert far.max() <= 1, f"{(far > 1).sum()} of {far.size}, the worst {far.max():.3g} times what is allowed"


def set_values(c, b, pos, block, x):
    """Block `block` of the value row at a position, of every kv head, holds x."""
    page, slot = c.place(b, pos)
    c.v[page, :, slot, block * BLOCK:(block + 1) * BLOCK] = host.quantize(np.asarray(x, dtype=np.float32))


WIDE = {"from zero": np.linspace(0, 150000, 32), "high": np.linspace(60000, 72000, 32), "both": np.linspace(-60000, 390000, 32),
        "largest": np.linspace(65000, 1040000, 32)}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", WIDE)
@pytest.mark.parametrize("heads,head_dim,tokens", [(4, 64, 1), (8, 128, 1), (4, 128, 5), (2, 64, 6), (12, 256, 1)])
def test_value_blocks_beyond_half_precision(gpu, kind, heads, head_dim, tokens):
    """A value block whose step and least value are fp16 numbers, but whose middle is not, is read as what it says by the tokens that see it, and does not reach the
    others: those before it, and those whose window has passed it although it lies in the same 32 keys as some that they see."""
    rng = np.random.default_rng(head_dim + tokens)
    for at, window in ((70, 0), (89, 0), (64, 24), (2, 0)):
        c = random_cache(rng, 2, head_dim, 16, [90])
        set_values(c, 0, at, 1, WIDE[kind])
        assert np.isfinite(host.values(c.v[c.place(0, at)[0], :, at % 16])).all()
        q = rng.standard_normal((tokens, heads * head_dim)).astype(np.float32)
        got = Device(gpu, c).attention(q, tokens, heads, window)
        assert np.isfinite(got).all()
        within(got, *c.attention_weighed(q, tokens, heads, window))


@pytest.mark.gpu
@pytest.mark.parametrize("ratio", [13, 18, 26])
@pytest.mark.parametrize("heads,head_dim,tokens", [(4, 64, 1), (8, 128, 1), (4, 128, 5), (2, 96, 6), (12, 256, 1)])
def test_value_blocks_of_very_different_steps(gpu, heads, head_dim, tokens, ratio):
    """Steps of one channel block, of one key that has next to no weight, and of one key that only the last token sees, are 2^ratio times those of the rest: what is made of the rest
    is as exact as without them."""
    rng = np.random.default_rng(head_dim + ratio)
    low = np.float32(2.0 ** -12)
    for kind in ("block", "key", "last"):
        c = random_cache(rng, 2, head_dim, 16, [100])
        for pos in range(100):
            page, slot = c.place(0, pos)
            c.v[page, :, slot] = host.quantize(rng.standard_normal((2, head_dim)).astype(np.float32) * low)
            if kind == "block":
                set_values(c, 0, pos, 0, rng.standard_normal(32) * low * 2.0 ** ratio)
        q = (rng.standard_normal((tokens, heads * head_dim)) * 0.05).astype(np.float32)
        large = host.quantize(rng.standard_normal((2, head_dim)).astype(np.float32) * low * np.float32(2.0 ** ratio))
        if kind == "key":                                       # its scores are -60 and less: all queries have a part along it
            q.reshape(tokens, heads, head_dim)[..., 0] = 2.0
            page, slot = c.place(0, 9)
            k = np.zeros((2, head_dim), dtype=np.float32)
            k[:, 0] = -30 * np.sqrt(head_dim)
            c.k[page, :, slot], c.v[page, :, slot] = host.quantize(k), large
        elif kind == "last":
            page, slot = c.place(0, 99)
            c.v[page, :, slot] = large
        within(Device(gpu, c).attention(q, tokens, heads), *c.attention_weighed(q, tokens, heads))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,head_dim,tokens,window", [(4, 64, 1, 0), (8, 128, 1, 0), (16, 128, 3, 0), (8, 256, 2, 40)])
def test_value_blocks_of_all_magnitudes(gpu, heads, head_dim, tokens, window):
    """Each block of each key has a magnitude of its own between 2^-20 and 2^15, some are all one number, some all zero."""
    rng = np.random.default_rng(heads + head_dim)
    c = random_cache(rng, 2, head_dim, 16, [150, 31])
    for b, n in enumerate(c.lens):
        for pos in range(int(n)):
            x = rng.standard_normal((2, head_dim // 32, 32)) * 2.0 ** rng.integers(-20, 16, (2, head_dim // 32, 1))
            x = np.where(rng.random((2, head_dim // 32, 1)) < 0.1, x[..., :1], x)
            x = np.where(rng.random((2, head_dim // 32, 1)) < 0.1, 0, x)
            page, slot = c.place(b, pos)
            c.v[page, :, slot] = host.quantize(x.reshape(2, head_dim).astype(np.float32))
    q = (rng.standard_normal((2 * tokens, heads * head_dim)) * 0.5).astype(np.float32)
    within(Device(gpu, c).attention(q, tokens, heads, window), *c.attention_weighed(q, tokens, heads, window))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,head_dim,page_tokens,lens,tokens,window,columns", [
    (16, 2, 128, 16, [150, 33, 0, 700] + [(29 * i) % 90 for i in range(16)], 1, 0, 960),      # four CTAs an SM
    (7, 1, 128, 64, [300, 64], 1, 50, 1), (24, 3, 64, 48, [200, 5], 3, 0, 1), (9, 1, 96, 16, [70], 2, 33, 1), (4, 2, 192, 16, [90, 200], 4, 0, 1), (3, 3, 192, 32, [130], 1, 0, 1),
    (20, 2, 256, 16, [60, 40], 2, 0, 1), (4, 1, 128, 32, [2500], 1, 0, 1), (6, 1, 64, 16, [40], 40, 7, 1)])
def test_magnitudes_in_every_form(gpu, heads, kv_heads, head_dim, page_tokens, lens, tokens, window, columns):
    """The same for every number of rows and channels, with pages missing, a page that does not exist and windows; steps of neighbours 2^-24 to 2^15 apart, some blocks no numbers."""
    rng = np.random.default_rng(heads + 7 * head_dim)
    c = random_cache(rng, kv_heads, head_dim, page_tokens, lens, extra_columns=columns, hole=True)
    for b, n in enumerate(lens):
        for pos in range(n):
            at = c.place(b, pos)
            if not at:
                continue
            x = rng.standard_normal((kv_heads, head_dim // 32, 32)) * 2.0 ** rng.choice([-20, -13, -12, 0, 1, 2, 2, 2, 13], (kv_heads, head_dim // 32, 1))
            c.v[at[0], :, at[1]] = host.quantize((x + 10.0 * rng.standard_normal(x.shape[:2] + (1,)) * (rng.random(x.shape[:2] + (1,)) < 0.1)).reshape(kv_heads, head_dim).astype(np.float32))
            if rng.random() < 0.004:
                c.v[at[0], :, at[1], :4] = 255
    q = (rng.standard_normal((len(lens) * tokens, heads * head_dim)) * 0.3).astype(np.float32)
    within(Device(gpu, c).attention(q, tokens, heads, window), *c.attention_weighed(q, tokens, heads, window))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,head_dim,tokens", [(4, 64, 1), (8, 128, 1), (4, 128, 5), (16, 64, 1)])
def test_long_sequences_of_distinct_rows(gpu, heads, head_dim, tokens):
    """70001 rows, no two alike, against torch in 64 bits: 3e-6 of the result's norm, a dozen roundings to the 22 bits of two fp16 pieces."""
    rng, n, pt = np.random.default_rng(heads + head_dim), 70001, 64
    pages = -(-n // pt)
    c = Cache(1, head_dim, pt, pages, rng.permutation(pages)[None], [n])
    for pool in (c.k, c.v):
        pool[:] = host.quantize(rng.standard_normal((pages, 1, pt, head_dim)).astype(np.float32))
    q = rng.standard_normal((tokens, heads * head_dim)).astype(np.float32)
    got = Device(gpu, c).attention(q, tokens, heads)
    k, v = (up(host.values(pool[c.table[0], 0]).reshape(-1, head_dim)[:n]) for pool in (c.k, c.v))
    score = (up(q.astype(np.float64)).view(tokens, heads, head_dim) @ k.T) / np.sqrt(head_dim)
    score.masked_fill_(torch.arange(n, device="cuda") > torch.arange(n - tokens, n, device="cuda").view(-1, 1, 1), -torch.inf)
    want = (torch.softmax(score, -1) @ v).reshape(tokens, -1).cpu().numpy()
    assert np.linalg.norm(got - want) <= 3e-6 * np.linalg.norm(want), np.linalg.norm(got - want) / np.linalg.norm(want)
