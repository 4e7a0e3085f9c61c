"""The paged 4-bit KV cache and the attention that reads it, as cases that can be timed and compared.

  attention  one or several new tokens of each sequence over a cache of Q4_1 rows in pages
  rows       new keys and values go into such a cache and are read back as fp32 (what a prompt's own attention is given)
  branch     sequences are forked (or not) and then grow by some tokens: pages are shared, copied on write and taken from the free ones
  compact    the pages in use move to the front of the pool

A cache row is head_dim / 32 blocks of 20 bytes: fp16 d, fp16 m, 16 bytes whose low nibbles are the codes of values 0..15 and whose high
nibbles those of values 16..31; a value is d * code + m.  A page holds page_tokens rows of every kv head, [kv heads][page_tokens][row]."""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

BLOCK = 20


def listed():
    return [
        # a chat with a small model that has just begun: latency of one call
        dict(name="attention 14/2x64 77", kind="attention", heads=14, kv_heads=2, head_dim=64, batch=1, tokens=1, longest=77, shortest=77, page=16, window=0),
        # an assistant's single conversation on an 8B model
        dict(name="attention 32/8x128 4096", kind="attention", heads=32, kv_heads=8, head_dim=128, batch=1, tokens=1, longest=4096, shortest=4096, page=64, window=0),
        # a server's decode step of the 70B shape: 32 conversations of different lengths
        dict(name="attention 64/8x128 batch 32", kind="attention", heads=64, kv_heads=8, head_dim=128, batch=32, tokens=1, longest=4096, shortest=2011, page=64, window=0),
        # the check of five drafted tokens for each of 16 sequences
        dict(name="attention 5 drafts batch 16", kind="attention", heads=32, kv_heads=8, head_dim=128, batch=16, tokens=5, longest=8190, shortest=301, page=32, window=0),
        # documents: four very long sequences
        dict(name="attention 64/8x128 131072", kind="attention", heads=64, kv_heads=8, head_dim=128, batch=4, tokens=1, longest=131072, shortest=129001, page=256, window=0),
        # a later turn of a conversation: 129 tokens behind 1024, windowed
        dict(name="attention 129 after 1024", kind="attention", heads=32, kv_heads=8, head_dim=128, batch=1, tokens=129, longest=1153, shortest=1153, page=64, window=1000),
        # the row that a decode step adds to each of 32 sequences
        dict(name="rows 1 x 32", kind="rows", kv_heads=8, head_dim=128, batch=32, tokens=1, longest=4096, shortest=2011, page=64),
        # prompts of four sequences
        dict(name="rows 2048 x 4", kind="rows", kv_heads=8, head_dim=128, batch=4, tokens=2048, longest=2500, shortest=2048, page=64),
        # a decode step's turn of the page tables: every sequence one token longer
        dict(name="branch step batch 32", kind="branch", kv_heads=2, head_dim=64, layers=24, batch=32, parents=32, add=1, longest=1000, shortest=33, page=16, pages=2500),
        # eight prompts of the 70B shape, each continued in six ways
        dict(name="branch 8 into 48", kind="branch", kv_heads=8, head_dim=128, layers=80, batch=48, parents=8, add=3, longest=500, shortest=400, page=64, pages=512),
        # defragmenting a small model's pool
        dict(name="compact 24 layers", kind="compact", kv_heads=2, head_dim=64, layers=24, batch=40, shared=0, longest=200, shortest=20, page=16, pages=512),
        # and the 70B shape's, some prompts shared
        dict(name="compact 80 layers", kind="compact", kv_heads=8, head_dim=128, layers=80, batch=48, shared=2, longest=600, shortest=100, page=64, pages=400),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "rows", "branch", "compact"])
    kv_heads, head_dim, page = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 96, 128, 128, 256]), rng.choice([16, 32, 64, 128, 256, 48])
    if kind == "attention":
        batch = _log(rng, 1, 64)
        tokens = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 200)])
        heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 12])
        longest = _log(rng, 1, max(2, min(131072, 5.0e8 / (batch * kv_heads * head_dim * BLOCK / 16))))
        shortest = longest if rng.random() < 0.3 else _log(rng, 1, longest)
        case = dict(kind=kind, heads=heads, kv_heads=kv_heads, head_dim=head_dim, batch=batch, tokens=tokens, longest=longest, shortest=shortest,
                    page=page, window=0 if rng.random() < 0.7 else _log(rng, 1, max(2, longest)))
        while work(case)["flops"] > 1.6e10:
            case |= dict(longest=-(-case["longest"] // 2), shortest=-(-case["shortest"] // 2), tokens=-(-case["tokens"] // 2))
        return case
    if kind == "rows":
        batch = _log(rng, 1, 64)
        tokens = _log(rng, 1, max(1, 8192 // batch))
        longest = tokens + _log(rng, 1, 2000)
        return dict(kind=kind, kv_heads=kv_heads, head_dim=head_dim, batch=batch, tokens=tokens, longest=longest, shortest=_log(rng, 1, longest), page=page)
    layers, batch, longest = rng.choice([2, 8, 24, 32]), _log(rng, 2, 48), _log(rng, 2, 40 * page)
    case = dict(kind=kind, kv_heads=kv_heads, head_dim=head_dim, layers=layers, batch=batch, longest=longest, shortest=_log(rng, 1, longest), page=page)
    used = sum(-(-n // page) for n in _lengths(case))
    spare = (1.0e9 / (2 * layers * kv_heads * page * head_dim * BLOCK / 32))
    if kind == "branch":
        case |= dict(parents=rng.randint(1, batch), add=_log(rng, 1, 2 * page))
        return case | dict(pages=used + sum(1 + -(-case["add"] // page) for _ in range(batch)) + batch + rng.randint(0, max(1, int(min(spare, 4 * used)))))
    return case | dict(shared=rng.choice([0, 1, 3]), pages=used + rng.randint(0, max(1, int(min(spare, 2 * used)))))


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """Tokens in each sequence: the longest first, the others spread down to the shortest."""
    span = case["longest"] - case["shortest"] + 1
    return [case["longest"] - (i * 2654435761 >> 7) % span for i in range(case["batch"])]


def _page_bytes(case):
    return case["kv_heads"] * case["page"] * case["head_dim"] // 32 * BLOCK


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    return _prepare_pool(case, seed) if case["kind"] in ("branch", "compact") else _prepare_rows(case, seed)


def _prepare_rows(case, seed):
    g = _generator(seed)
    batch, page, hkv, hd = case["batch"], case["page"], case["kv_heads"], case["head_dim"]
    lens = _lengths(case)
    stride = -(-case["longest"] // page) + 1
    used = [-(-n // page) for n in lens]
    pages = sum(used) + 2
    order = np.random.RandomState(seed & 0x7FFFFFFF).permutation(pages)
    table = np.full((batch, stride), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    s = dict(case=case, batch=batch, page=page, kv_heads=hkv, head_dim=hd, tokens=case["tokens"], stride=stride, pages=pages, longest=case["longest"],
             table=torch.from_numpy(table).cuda(), lens=_ints(lens))
    rows = (batch * case["tokens"], hkv * hd)
    if case["kind"] == "rows":
        # a layer's fused projection: keys and values are parts of its rows
        qkv = torch.randn(rows[0], 2 * rows[1], device="cuda", generator=g)
        s |= dict(k=qkv[:, :rows[1]], v=qkv[:, rows[1]:], k_back=torch.empty(rows, device="cuda"), v_back=torch.empty(rows, device="cuda"),
                  k_pages=torch.zeros(pages, _page_bytes(case), dtype=torch.uint8, device="cuda"), v_pages=torch.zeros(pages, _page_bytes(case), dtype=torch.uint8, device="cuda"))
    else:
        # keys have a few channels of large values, as trained models' do; what is in pages that nobody holds is no number
        spread = torch.ones(hkv, 1, hd, device="cuda")
        spread[:, :, ::37] = 4.0
        for name in ("k_pages", "v_pages"):
            x = torch.randn(pages, hkv, page, hd, device="cuda", generator=g)
            if name == "k_pages":
                x *= spread
            s[name] = _quantize(x).view(pages, -1)
            del x
            s[name][torch.from_numpy(order[at:]).cuda()] = 255
        s |= dict(window=case["window"], heads=case["heads"], q=torch.randn(rows[0], case["heads"] * hd, device="cuda", generator=g),
                  out=torch.empty(rows[0], case["heads"] * hd, device="cuda"))
    if own:
        s["lib"] = _lib()
        if case["kind"] == "attention":
            n = s["lib"].ckb200_attention_q4cache_workspace_bytes(batch, case["tokens"], case["heads"], hkv, hd)
            s["workspace"] = torch.empty(max(1, n), dtype=torch.uint8, device="cuda")
    return s


def _live_pages(case):
    """Which pages are in use, how many of them each sequence shares with the one before it, and the lengths: the same for every seed."""
    lens = _lengths(case)
    used = [-(-n // case["page"]) for n in lens]
    shared = [min(case.get("shared", 0), used[b], used[b - 1]) if b % 2 else 0 for b in range(case["batch"])]
    # a shared page is full
    shared = [min(n, lens[b] // case["page"], lens[b - 1] // case["page"]) if n else 0 for b, n in enumerate(shared)]
    live = sum(used) - sum(shared)
    return sorted(random.Random(live * 1000003 + case["pages"]).sample(range(case["pages"]), live)), shared, lens


def _prepare_pool(case, seed):
    g = _generator(seed)
    batch, page = case["batch"], case["page"]
    live, shared, lens = _live_pages(case)
    order = np.random.RandomState(seed & 0x7FFFFFFF).permutation(np.array(live, dtype=np.int32))
    add = case.get("add", 0)
    stride = -(-(case["longest"] + add) // page) + 1
    table = np.full((batch, stride), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(lens):
        n = -(-n // page)
        table[b, :shared[b]] = table[b - 1, :shared[b]]
        table[b, shared[b]:n] = order[at:at + n - shared[b]]
        at += n - shared[b]
    refs = np.bincount(table[table >= 0], minlength=case["pages"]).astype(np.int32)
    start = torch.from_numpy(np.concatenate([table.ravel(), np.array(lens, dtype=np.int32), refs])).cuda()
    work = torch.empty_like(start)
    planes = 2 * case["layers"]
    s = dict(case=case, batch=batch, page=page, stride=stride, pages=case["pages"], planes=planes, page_bytes=_page_bytes(case), start=start, work=work,
             table=work[:batch * stride].view(batch, stride), lens=work[batch * stride:batch * stride + batch], refs=work[batch * stride + batch:],
             pool=torch.randint(-2**31, 2**31 - 1, (planes, case["pages"], _page_bytes(case) // 4), dtype=torch.int32, device="cuda", generator=g))
    if case["kind"] == "branch":
        parent = [b % case["parents"] for b in range(batch)]
        s |= dict(parent=_ints(parent), new_lens=_ints([lens[p] + add for p in parent]), status=torch.empty(batch, dtype=torch.int32, device="cuda"))
    else:
        s["live"] = torch.empty(1, dtype=torch.int32, device="cuda")
    if own:
        s["lib"] = _lib()
        n = s["lib"].ckb200_kv_pages_workspace_bytes(batch, stride, case["pages"])
        s["workspace"] = torch.empty(max(1, n), dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    kind = s["case"]["kind"]
    if kind == "attention":
        return _attention_own(s) if own else _attention(s)
    if kind == "rows":
        return _rows_own(s) if own else _rows(s)
    s["work"].copy_(s["start"])
    if kind == "branch":
        if own:
            _branch_own(s)
        else:
            _fork(s)
            _resize(s)
        return dict(pool=s["pool"], table=s["table"], lens=s["lens"], refs=s["refs"], status=s["status"])
    if own:
        _compact_own(s)
    else:
        _compact(s)
    return dict(pool=s["pool"], table=s["table"], refs=s["refs"], live=s["live"])


# ---- the framework's calls

_bound = None


def _lib():
    global _bound
    if _bound is None:
        import __graft_entry__ as graft
        torch.cuda.init()
        torch.cuda.current_stream()
        pkg = graft.load_package()
        lib = pkg.load_lib()
        pkg.cache_api.bind_cache_api(lib)
        if lib.ckb200_init(0) != 0:
            raise RuntimeError(lib.ckb200_last_error_message().decode())
        _bound = lib
    return _bound


def _stream():
    return torch.cuda.current_stream().cuda_stream or 1      # 1: the handle of the default stream, where NULL means the library's own


def _ok(s, rc):
    if rc:
        raise RuntimeError((s["lib"].ckb200_last_error_message() or b"call failed").decode())


def _attention_own(s):
    _ok(s, s["lib"].ckb200_dev_attention_q4cache(
        s["q"].data_ptr(), s["heads"] * s["head_dim"], s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["out"].data_ptr(), s["heads"] * s["head_dim"],
        s["table"].data_ptr(), s["stride"], s["lens"].data_ptr(), s["batch"], s["tokens"], s["pages"], s["page"], s["heads"], s["kv_heads"], s["head_dim"], s["window"],
        s["workspace"].data_ptr(), s["workspace"].numel(), _stream()))
    return s["out"]


def _rows_own(s):
    n, where = s["kv_heads"] * s["head_dim"], (s["table"].data_ptr(), s["stride"], s["lens"].data_ptr(), s["batch"], s["tokens"], s["pages"], s["page"], s["kv_heads"], s["head_dim"])
    st = _stream()
    _ok(s, s["lib"].ckb200_dev_kv_cache_store_q4(s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), 2 * n, 2 * n, *where, st))
    _ok(s, s["lib"].ckb200_dev_kv_cache_load_q4(s["k_back"].data_ptr(), s["v_back"].data_ptr(), n, n, s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), *where, st))
    return dict(k=s["k_back"], v=s["v_back"])


def _branch_own(s):
    st, ws = _stream(), (s["workspace"].data_ptr(), s["workspace"].numel())
    _ok(s, s["lib"].ckb200_dev_kv_pages_fork(s["table"].data_ptr(), s["stride"], s["lens"].data_ptr(), s["refs"].data_ptr(), s["parent"].data_ptr(), s["batch"], s["pages"], s["page"], *ws, st))
    _ok(s, s["lib"].ckb200_dev_kv_pages_resize(s["table"].data_ptr(), s["stride"], s["lens"].data_ptr(), s["refs"].data_ptr(), s["new_lens"].data_ptr(), s["batch"], s["pages"], s["page"],
                                               s["pool"].data_ptr(), s["planes"], s["pages"] * s["page_bytes"], s["page_bytes"], s["status"].data_ptr(), *ws, st))


def _compact_own(s):
    _ok(s, s["lib"].ckb200_dev_kv_pages_compact(s["table"].data_ptr(), s["stride"], s["lens"].data_ptr(), s["refs"].data_ptr(), s["batch"], s["pages"], s["page"],
                                                s["pool"].data_ptr(), s["planes"], s["pages"] * s["page_bytes"], s["page_bytes"], s["live"].data_ptr(),
                                                s["workspace"].data_ptr(), s["workspace"].numel(), _stream()))


# ---- plain forms

def _quantize(x):
    """fp32 [..., n * 32] -> uint8 [..., n * 20]."""
    x = x.view(*x.shape[:-1], -1, 32)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m, d = low.half(), ((high - low) / torch.full_like(low, 15)).half()      # a division: by a number torch would multiply with its inverse
    inverse = torch.where(d > 0, 1 / d.float(), torch.zeros_like(low))
    code = torch.floor((x - m.float()) * inverse + 0.5).clamp_(0, 15).to(torch.uint8)
    qs = code[..., :16] | (code[..., 16:] << 4)
    return torch.cat([d.view(torch.uint8), m.view(torch.uint8), qs], -1).flatten(-2)


def _values(rows):
    """uint8 [..., n * 20] -> fp32 [..., n * 32]."""
    blocks = rows.unflatten(-1, (-1, BLOCK))
    dm = blocks[..., :4].contiguous().view(torch.float16).float()
    qs = blocks[..., 4:]
    code = torch.cat([qs & 15, qs >> 4], -1).float()
    return (code * dm[..., :1] + dm[..., 1:]).flatten(-2)


def _cached(s, pages):
    """The rows of every sequence, [batch, kv heads, tokens, bytes], for as many pages as the longest has."""
    n = -(-s["longest"] // s["page"])
    ids = s["table"][:, :n].clamp(min=0).long()
    rows = pages.view(s["pages"], s["kv_heads"], s["page"], -1)[ids]
    return rows.transpose(1, 2).flatten(2, 3)


def _attention(s):
    b, t, hkv, hd, group = s["batch"], s["tokens"], s["kv_heads"], s["head_dim"], s["heads"] // s["kv_heads"]
    k = _values(_cached(s, s["k_pages"]))
    key = torch.arange(k.shape[2], device="cuda")
    at = s["lens"].view(b, 1, 1) - t + torch.arange(t, device="cuda").view(1, t, 1)
    seen = key <= at
    if s["window"]:
        seen &= key > at - s["window"]
    q = s["q"].view(b, t, hkv, group, hd).permute(0, 2, 1, 3, 4).reshape(b, hkv, t * group, hd)
    score = (q @ k.transpose(-1, -2)).view(b, hkv, t, group, -1) * (1 / math.sqrt(hd))
    del k
    score.masked_fill_(~seen.view(b, 1, t, 1, -1), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    v = _values(_cached(s, s["v_pages"])).masked_fill_(~seen.any(1).view(b, 1, -1, 1), 0.0)
    out = (p.view(b, hkv, t * group, -1) @ v).view(b, hkv, t, group, hd) / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(0, 2, 1, 3, 4).reshape(b * t, -1)


def _rows(s):
    b, t, page, hkv = s["batch"], s["tokens"], s["page"], s["kv_heads"]
    at = (s["lens"].view(b, 1) - t + torch.arange(t, device="cuda")).view(-1).long()
    row = torch.arange(b, device="cuda").repeat_interleave(t)
    there = at >= 0
    at = at.clamp(min=0)
    ids, slot = s["table"][row, at // page].long(), at % page
    # rows before a sequence's first token have no place: they go to a page that nobody holds
    held = torch.zeros(s["pages"], dtype=torch.bool, device="cuda").index_fill_(0, s["table"].clamp(min=0).view(-1).long(), True)
    ids = torch.where(there, ids, torch.argmin(held.to(torch.int32)))
    back = []
    for x, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
        pool = pages.view(s["pages"], hkv, page, -1)
        pool[ids, :, slot] = _quantize(x.reshape(b * t, hkv, -1))
        back.append(_values(pool[ids, :, slot]).masked_fill_(~there.view(-1, 1, 1), 0.0).flatten(1))
    return dict(k=back[0], v=back[1])


def _fork(s):
    table, lens, parent = s["table"], s["lens"], s["parent"].long()
    self = torch.arange(s["batch"], device="cuda")
    source = torch.where((parent >= 0) & (parent < s["batch"]), parent, self)
    new, changed = table[source], source != self
    one = torch.ones_like(table)
    s["refs"].index_add_(0, new.clamp(min=0).view(-1), (one * (changed.view(-1, 1) & (new >= 0))).view(-1))
    s["refs"].index_add_(0, table.clamp(min=0).view(-1), (-one * (changed.view(-1, 1) & (table >= 0))).view(-1))
    lens.copy_(lens[source])
    table.copy_(new)


def _resize(s):
    """For pools with room for everything that is asked."""
    table, lens, refs, page = s["table"], s["lens"], s["refs"], s["page"]
    new = torch.where(s["new_lens"] < 0, lens, s["new_lens"])
    have, need = (lens + page - 1) // page, (new + page - 1) // page
    column = torch.arange(s["stride"], device="cuda")
    gone = (column >= need.view(-1, 1)) & (column < have.view(-1, 1))
    refs.index_add_(0, table.clamp(min=0).view(-1), -gone.to(torch.int32).view(-1))
    table.masked_fill_(gone, -1)
    each = torch.arange(s["batch"], device="cuda")
    column_of = (lens - 1).clamp(min=0).long() // page
    last = table[each, column_of]
    partial = (new > lens) & (lens % page != 0)
    same = (last.view(-1, 1) == last.view(1, -1)) & partial.view(1, -1) & (each.view(-1, 1) > each.view(1, -1))
    own_copy = partial & (refs[last.clamp(min=0).long()] - same.sum(1) > 1)
    wanted = own_copy.long() + (need - have).clamp(min=0)
    first = torch.cumsum(wanted, 0) - wanted
    free = torch.nonzero(refs == 0).view(-1)
    src, dst = last[own_copy].long(), free[first[own_copy]]
    s["pool"][:, dst] = s["pool"][:, src]
    refs.index_add_(0, src, -torch.ones_like(src, dtype=torch.int32))
    table[each[own_copy], column_of[own_copy]] = dst.to(torch.int32)
    fresh = (column >= have.view(-1, 1)) & (column < need.view(-1, 1))
    table[fresh] = free[((first + own_copy.long() - have).view(-1, 1) + column)[fresh]].to(torch.int32)
    refs[free[:wanted.sum()]] = 1
    lens.copy_(new)
    s["status"].zero_()


def _compact(s):
    table, refs, pool = s["table"], s["refs"], s["pool"]
    used = refs > 0
    count = int(used.sum())
    src, dst = torch.nonzero(used[count:]).view(-1) + count, torch.nonzero(~used[:count]).view(-1)
    place = torch.arange(s["pages"], dtype=torch.int32, device="cuda")
    place[src] = dst.to(torch.int32)
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()], table))
    pool[:, dst] = pool[:, src]
    refs[dst] = refs[src]
    refs[src] = 0
    s["live"].fill_(count)


# ------------------------------------------------------------------ what a pass has to do, and its results in 64 bits

def _seen(case):
    """(keys of the cache that are read, sum over queries of the keys that each sees)."""
    t, w, keys, pairs = case["tokens"], case["window"], 0, 0
    for n in _lengths(case):
        first = max(0, max(0, n - t) - w + 1) if w else 0
        keys += n - first
        for i in range(t):
            at = n - t + i
            pairs += max(0, at + 1) if not w else max(0, min(w, at + 1))
    return keys, pairs


def work(case):
    if case["kind"] == "attention":
        keys, pairs = _seen(case)
        q = case["batch"] * case["tokens"] * case["heads"] * case["head_dim"]
        return dict(bytes=keys * 2 * case["kv_heads"] * case["head_dim"] // 32 * BLOCK + 8 * q, flops=4 * pairs * case["heads"] * case["head_dim"])
    if case["kind"] == "rows":
        n = 2 * sum(min(k, case["tokens"]) for k in _lengths(case)) * case["kv_heads"] * case["head_dim"]
        return dict(bytes=2 * (4 * n + n // 32 * BLOCK), flops=8 * n)
    planes, lens = 2 * case["layers"], _lengths(case)
    entries = sum(-(-n // case["page"]) for n in lens)
    if case["kind"] == "compact":
        live = _live_pages(case)[0]
        moved = sum(p >= len(live) for p in live)
        return dict(bytes=2 * moved * planes * _page_bytes(case) + 8 * (entries + case["pages"]), flops=0)
    sharers = [0] * case["parents"]
    for b in range(case["batch"]):
        sharers[b % case["parents"]] += lens[b % case["parents"]] % case["page"] != 0
    copied = sum(max(0, n - 1) for n in sharers)
    return dict(bytes=2 * copied * planes * _page_bytes(case) + 8 * entries + 4 * case["pages"] + 16 * case["batch"], flops=0)


def exact(case, seed):
    if case["kind"] in ("branch", "compact"):
        return None
    s = prepare(case, seed)
    b, t, page, hkv, hd = s["batch"], s["tokens"], s["page"], s["kv_heads"], s["head_dim"]
    lens = _lengths(case)
    if case["kind"] == "rows":
        # which code a value gets is settled by the quantiser's fp32 steps, as with the other block formats; the value that it stands for is not
        found = {}
        for name in ("k", "v"):
            x = s[name].cpu().numpy().reshape(-1, 32)
            low, span = x.min(1), x.max(1) - x.min(1)
            m, d = low.astype(np.float16), (span / np.float32(15)).astype(np.float16)
            step = d.astype(np.float32)
            inverse = np.divide(np.float32(1), step, out=np.zeros_like(step), where=step > 0)
            code = np.trunc(np.clip((x - m.astype(np.float32)[:, None]) * inverse[:, None] + np.float32(0.5), 0, 15))
            y = torch.from_numpy(code.astype(np.float64) * d.astype(np.float64)[:, None] + m.astype(np.float64)[:, None]).cuda().view(b, t, hkv * hd)
            for i, n in enumerate(lens):
                y[i, :max(0, t - n)] = 0
            found[name] = y.reshape(b * t, hkv * hd)
        return found
    out = torch.zeros(b, t, case["heads"], hd, dtype=torch.float64, device="cuda")
    query = s["q"].double().view(b, t, case["heads"], hd)
    table = s["table"].tolist()
    group = case["heads"] // hkv
    for i, n in enumerate(lens):
        ids = torch.tensor(table[i][:-(-n // page)], device="cuda")
        lo = max(0, n - t)
        for h in range(hkv):
            kv = []
            for pages in (s["k_pages"], s["v_pages"]):
                raw = pages.view(s["pages"], hkv, page, hd // 32, BLOCK)[ids, h].reshape(-1, hd // 32, BLOCK)[:n]
                d, m = raw[..., 0:2].contiguous().view(torch.float16).double(), raw[..., 2:4].contiguous().view(torch.float16).double()
                kv.append(torch.cat([(raw[..., 4:] % 16).double(), torch.div(raw[..., 4:], 16, rounding_mode="floor").double()], -1).mul_(d).add_(m).reshape(n, hd))
            pos = torch.arange(lo, n, device="cuda").view(-1, 1, 1)
            keys = torch.arange(n, device="cuda").view(1, 1, -1)
            hidden = keys > pos
            if case["window"]:
                hidden = hidden | (keys <= pos - case["window"])
            score = torch.einsum("tgd,nd->tgn", query[i, t - (n - lo):, h * group:(h + 1) * group], kv[0]) / math.sqrt(hd)
            out[i, t - (n - lo):, h * group:(h + 1) * group] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ kv[1]
    return out.view(b * t, -1)
