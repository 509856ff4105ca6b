"""The serving operators on the GPU against plain implementations in 64 bits
(tests/serve_oracle.py): the paged cache's append and read-back bit for bit,
attention within bounds derived from its number formats, the logits' rules bit
for bit; at the sizes, layouts and masks where they can go wrong."""
import math
import sys

import numpy as np
import pytest
import torch

from aps2026_amd import attention, serve
from tests import serve_oracle as oracle

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def note(msg):
    print(f"[gpu-case] {msg}", flush=True)
    sys.stdout.flush()


def f64(t):
    return t.detach().cpu().double().numpy()


def bits(t):
    return t.detach().cpu().contiguous().view({4: torch.int32, 2: torch.int16, 1: torch.uint8}[t.element_size()])


def make_cache(kind, pages, kv_heads, page, dim, dev, rng, garbage=False):
    """A cache of N(0, 1) values (garbage: NaN everywhere) and its float64 values."""
    shape = (pages, kv_heads, page, dim)
    if kind == "mxfp4":
        if garbage:
            t = [np.full((*shape[:3], dim // 2), 0x77, np.uint8), np.full((*shape[:3], dim // 32), 255, np.uint8)] * 2
        else:
            t = [a for _ in range(2) for a in oracle.mx_encode(rng.standard_normal(shape, dtype=np.float32))]
        kc, ks, vc, vs = (torch.from_numpy(a.copy()).to(dev) for a in t)
        return serve.PagedKvCache(kc, vc, ks, vs)
    dt = {"f32": F32, "bf16": BF16}[kind]
    x = [np.full(shape, np.nan, np.float32) if garbage else rng.standard_normal(shape, dtype=np.float32)
         for _ in range(2)]
    return serve.PagedKvCache(*(torch.from_numpy(a).to(dev, dt) for a in x))


def held(cache):
    """float64 k and v [pages, kv_heads, page, dim] of a cache."""
    if cache.dtype == serve.MXFP4:
        return [oracle.mx_values(c.cpu().numpy(), s.cpu().numpy())
                for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    return [f64(cache.k), f64(cache.v)]


# ---- append and read-back -----------------------------------------------------

APPEND = [
    # src, cache, q_heads, kv_heads, dim, page, rows, layout
    (F32, "bf16", 16, 4, 128, 16, 37, "plain"),
    (F32, "f32", 16, 4, 128, 16, 1, "plain"),
    (BF16, "bf16", 16, 4, 128, 64, 131, "fused"),
    (BF16, "mxfp4", 8, 8, 64, 32, 19, "fused"),
    (F32, "mxfp4", 16, 4, 128, 16, 67, "plain"),
    (F32, "mxfp4", 2, 1, 64, 256, 5, "odd"),
    (BF16, "bf16", 6, 2, 64, 128, 23, "odd"),
    (F32, "bf16", 5, 5, 128, 16, 8, "odd"),
    (F32, "f32", 24, 4, 64, 16, 9, "no_q"),
    (BF16, "mxfp4", 16, 4, 128, 16, 40, "in_place"),
]


@pytest.mark.parametrize("src,kind,qh,kvh,dim,page,rows,layout", APPEND)
def test_append_and_gather(gpu_device, src, kind, qh, kvh, dim, page, rows, layout):
    note(f"append {src} {kind} heads {qh}/{kvh} dim {dim} page {page} rows {rows} {layout}")
    dev = gpu_device
    rng = np.random.default_rng(rows * 7 + dim)
    pages, max_pos = -(-rows // page) + 2, 50
    cache = make_cache(kind, pages, kvh, page, dim, dev, rng)
    before = held(cache)
    widths = [qh * dim, kvh * dim, kvh * dim]
    if layout in ("fused", "in_place"):
        row = torch.from_numpy(rng.standard_normal((rows, sum(widths)), dtype=np.float32)).to(dev, src)
        q, k, v = row.split(widths, 1)
    else:
        pad = 3 if layout == "odd" else 0       # odd: rows and starts off 16 bytes
        q, k, v = (torch.from_numpy(rng.standard_normal((rows, w + pad), dtype=np.float32)).to(dev, src)[:, pad:]
                   for w in widths)
    x = [f64(t).reshape(rows, -1, dim) for t in (q, k, v)]
    cos, sin = attention.rope_table(max_pos, dim)
    pos = rng.integers(0, max_pos, rows).astype(np.int32)
    slots = rng.permutation(pages * page)[:rows].astype(np.int64)
    if rows > 6:
        pos[2], pos[3], pos[4] = max_pos, -1, 0                     # outside the table: unrotated
        slots[1], slots[5], slots[6] = -1, pages * page, 1 << 40    # padding: not written
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    q_out = q if layout == "in_place" else None
    got_q = serve.kv_append_gpu(cache, k, v, d(pos), d(slots), d(cos), d(sin), q=None if layout == "no_q" else q,
                                q_out=q_out)
    torch.cuda.synchronize()
    want = [oracle.rotate(x[0], pos, cos, sin), oracle.rotate(x[1], pos, cos, sin), x[2].astype(np.float32)]
    if layout == "no_q":
        assert got_q is None
    else:
        assert (got_q.data_ptr() == q.data_ptr()) == (layout == "in_place")
        assert torch.equal(bits(got_q), bits(torch.from_numpy(want[0]).to(src).view(rows, -1)))
    ok = (slots >= 0) & (slots < pages * page)
    at = slots[ok] // page, slots[ok] % page
    for which in (0, 1):
        rows_now = want[1 + which][ok]
        if kind == "mxfp4":
            expect = before[which].copy()
            expect[at[0], :, at[1]] = oracle.mx_values(*oracle.mx_encode(rows_now))
        else:
            expect = before[which].copy()
            expect[at[0], :, at[1]] = torch.from_numpy(rows_now).to({"f32": F32, "bf16": BF16}[kind]).double().numpy()
        assert np.array_equal(held(cache)[which], expect)
        for dt in (F32, BF16):
            got = serve.kv_gather_gpu(cache, d(slots), dt)[which]
            back = np.zeros((rows, kvh, dim))
            back[ok] = expect[at[0], :, at[1]]
            assert torch.equal(got.cpu().view(rows, kvh, dim), torch.from_numpy(back).to(dt))


def test_append_blocks_that_are_not_finite(gpu_device):
    """A block with an infinity or a NaN reads back as NaN, its neighbours as
    they are; zeros and the smallest values keep their scale."""
    dev, dim = gpu_device, 64
    x = np.ones((4, dim), np.float32)
    x[0, 3], x[1, 40], x[2, :32], x[3, 32:] = np.inf, np.nan, 0.0, 2.0 ** -126
    cache = serve.PagedKvCache.allocate(1, 16, 1, dim, "mxfp4", dev)
    slots = torch.arange(4, device=dev)
    pos = torch.full((4,), -1, dtype=torch.int32, device=dev)
    t = torch.from_numpy(x).to(dev)
    table = torch.zeros(1, dim // 2, device=dev)
    serve.kv_append_gpu(cache, t, t, pos, slots, table, table)
    for got in serve.kv_gather_gpu(cache, slots):
        want = x.copy()
        want[0, :32], want[1, 32:] = np.nan, np.nan
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)


def test_append_and_gather_of_nothing(gpu_device):
    cache = serve.PagedKvCache.allocate(2, 16, 2, 64, BF16, gpu_device)
    e = torch.empty(0, 128, dtype=BF16, device=gpu_device)
    i32, i64 = (torch.empty(0, dtype=t, device=gpu_device) for t in (torch.int32, torch.int64))
    table = torch.zeros(1, 32, device=gpu_device)
    assert serve.kv_append_gpu(cache, e, e, i32, i64, table, table, q=e).shape == (0, 128)
    assert serve.kv_gather_gpu(cache, i64)[0].shape == (0, 128)


# ---- attention ------------------------------------------------------------------

# q type, cache, q_heads, kv_heads, dim, page
LAYOUTS = [
    (F32, "f32", 16, 4, 128, 16), (F32, "bf16", 16, 4, 128, 16), (F32, "mxfp4", 16, 4, 128, 16),
    (BF16, "bf16", 16, 4, 128, 64), (BF16, "mxfp4", 16, 4, 128, 32),
    (F32, "f32", 2, 2, 64, 32), (F32, "bf16", 6, 2, 64, 256), (F32, "mxfp4", 10, 2, 64, 16),
    (BF16, "bf16", 5, 5, 64, 16), (BF16, "mxfp4", 20, 1, 64, 128), (BF16, "bf16", 24, 1, 128, 16),
]

# new tokens and cached lengths of each sequence, window, sinks
SHAPES = {
    "one": ([1], [1], 2047, 4),
    "steps": ([1, 1, 1, 1], [1, 33, 130, 64], 2047, 0),
    "window": ([1, 1, 1], [200, 97, 20], 40, 5),
    "window_one": ([1, 3], [70, 35], 1, 0),
    "sinks_all": ([2, 1], [50, 120], 16, 1000),
    "guesses": ([5, 3, 9], [90, 3, 161], 64, 4),
    "empty": ([0, 2, 0, 4, 1], [0, 5, 31, 2, 0], 16, 2),      # more queries than keys, no keys, no queries
    "chunk": ([77, 40], [77, 200], 2047, 0),
    "mixed": ([1, 90, 0, 2, 1, 1, 3, 1, 1, 1], [70, 90, 4, 2, 300, 33, 3, 1, 0, 64], 2047, 1),
    "chunk_window": ([100, 33, 1], [150, 33, 90], 30, 7),
}


class Case:
    """A paged batch whose unused slots and pages hold NaN."""

    def __init__(self, dev, qt, kind, qh, kvh, dim, page, q_lens, kv_lens, seed=0, extra_rows=0):
        rng = np.random.default_rng(seed)
        self.dev, self.qt, self.qh, self.kvh, self.dim, self.page = dev, qt, qh, kvh, dim, page
        counts = [-(-n // page) for n in kv_lens]
        self.pages = sum(counts) + 2
        ids = rng.permutation(self.pages)
        self.table = np.full((len(q_lens), max(counts + [1])), -1, np.int32)
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.cache = make_cache(kind, self.pages, kvh, page, dim, dev, rng, garbage=True)
        full = make_cache(kind, self.pages, kvh, page, dim, dev, rng)
        live = torch.zeros(self.pages, page, dtype=torch.bool)
        for b, n in enumerate(kv_lens):
            for j in range(n):
                live[self.table[b, j // page], j % page] = True
        live = live[:, None, :, None].to(dev)
        for name in ("k", "v", "k_scale", "v_scale"):
            have = getattr(self.cache, name)
            if have is not None:
                have.copy_(torch.where(live, getattr(full, name), have))
        self.offs = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        self.kv_lens = np.asarray(kv_lens, np.int32)
        self.rows = int(self.offs[-1]) + extra_rows
        self.q = torch.from_numpy(rng.standard_normal((self.rows, qh * dim), dtype=np.float32)).to(dev, qt)
        self.max_q, self.max_kv = max(q_lens), max(kv_lens)

    def up(self, a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(self.dev)

    def run(self, window, sinks, scale=None, **kw):
        kw.setdefault("max_q_len", self.max_q)
        kw.setdefault("max_kv_len", self.max_kv)
        return serve.attention_paged_gpu(self.q, self.cache, self.up(self.offs), self.up(self.kv_lens),
                                         self.up(self.table), q_heads=self.qh, window=window, sinks=sinks,
                                         scale=scale, **kw)

    def check(self, got, window, sinks, scale=None):
        scale = 1 / math.sqrt(self.dim) if scale is None else scale
        k, v = held(self.cache)
        want, mag, prod, seen = oracle.attention(
            f64(self.q).reshape(self.rows, self.qh, self.dim), k, v, self.offs, self.kv_lens, self.table, self.page,
            self.qh, window, sinks, scale, self.pages)
        n = int(self.offs[-1])
        # weights of bf16 queries may be rounded to bf16 (8 bits), of fp32 ones to 24
        bound = oracle.attention_bound(want, mag, prod, seen, self.dim, self.qt, 24 if self.qt is F32 else 8)
        g = f64(got).reshape(self.rows, self.qh, self.dim)[:n]
        assert np.isfinite(g).all()
        off = np.abs(g - want[:n])
        worst = (off / bound[:n]).max() if n else 0.0
        note(f"  worst {worst:.3f} of the bound")
        assert worst <= 1.0


@pytest.mark.parametrize("qt,kind,qh,kvh,dim,page", LAYOUTS)
@pytest.mark.parametrize("shape", list(SHAPES))
def test_attention(gpu_device, qt, kind, qh, kvh, dim, page, shape):
    q_lens, kv_lens, window, sinks = SHAPES[shape]
    note(f"attention {qt} {kind} heads {qh}/{kvh} dim {dim} page {page} {shape}")
    c = Case(gpu_device, qt, kind, qh, kvh, dim, page, q_lens, kv_lens, seed=len(shape))
    c.check(c.run(window, sinks), window, sinks)


@pytest.mark.parametrize("qt,kind,dim", [(F32, "f32", 128), (F32, "bf16", 128), (F32, "mxfp4", 128),
                                         (BF16, "bf16", 128), (BF16, "mxfp4", 64), (BF16, "bf16", 64)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [1500]), ([1, 1], [3, 2100]), ([3], [1333])])
def test_attention_split(gpu_device, qt, kind, dim, q_lens, kv_lens):
    """Few rows and many keys: the key axis is split over workgroups."""
    note(f"attention split {qt} {kind} {q_lens} {kv_lens}")
    c = Case(gpu_device, qt, kind, 4, 1, dim, 16, q_lens, kv_lens, seed=3)
    need = __import__("aps2026_amd.capi", fromlist=["lib"]).lib().aps_attention_paged_workspace_size(
        c.cache._ref, c.rows, 4, len(q_lens), c.max_q, c.max_kv, 1 << 30, 0)
    assert need > 0
    c.check(c.run(1 << 30, 0), 1 << 30, 0)
    c.check(c.run(300, 9), 300, 9)


@pytest.mark.parametrize("qt,kind", [(F32, "bf16"), (F32, "mxfp4"), (BF16, "bf16"), (BF16, "mxfp4")])
@pytest.mark.parametrize("qh,kvh,dim,q_lens", [(3, 3, 64, [4, 1, 3]), (4, 2, 128, [2, 0, 1]), (6, 2, 128, [1, 1, 1]),
                                               (4, 1, 64, [1, 2, 1]), (7, 1, 128, [1, 1, 1]), (2, 1, 64, [4, 3, 1]),
                                               (5, 1, 64, [1, 1, 1]), (1, 1, 128, [8, 5, 2]), (9, 1, 64, [1, 1, 1])])
def test_attention_of_few_rows(gpu_device, qt, kind, qh, kvh, dim, q_lens):
    """1 to 9 rows under a key head, where terms of numbers stand beside rows;
    short, long and windowed, queries and keys of very different sizes."""
    note(f"few rows {qt} {kind} {qh}/{kvh} {dim} {q_lens}")
    c = Case(gpu_device, qt, kind, qh, kvh, dim, 16, q_lens, [9, 70, 1100], seed=12)
    c.check(c.run(1 << 30, 0), 1 << 30, 0)
    c.check(c.run(37, 3), 37, 3)
    c.q *= torch.exp2(torch.randint(-6, 3, c.q.shape, device=c.dev).float()).to(qt)
    c.check(c.run(1 << 30, 0), 1 << 30, 0)


@pytest.mark.parametrize("qt,kind", [(F32, "f32"), (F32, "bf16"), (F32, "mxfp4"), (BF16, "bf16"), (BF16, "mxfp4")])
@pytest.mark.parametrize("qh,kvh,dim,n,kv,window", [(4, 1, 64, 40, 900, 1 << 30), (2, 2, 128, 3, 900, 1 << 30),
                                                    (2, 1, 64, 30, 700, 333), (8, 1, 128, 2, 700, 250)])
def test_rows_computed_again(gpu_device, qt, kind, qh, kvh, dim, n, kv, window):
    """Long rows next to rows that see an infinite value keep their own."""
    note(f"again {qt} {kind} {qh}/{kvh} {dim} {n} {kv} {window}")
    c = Case(gpu_device, qt, kind, qh, kvh, dim, 16, [n], [kv], seed=21)
    j = kv - 2
    page, off = c.table[0, j // 16], j % 16
    if kind == "mxfp4":
        c.cache.v_scale[page, :, off] = 255
    else:
        c.cache.v[page, :, off] = -float("inf")
    got = f64(c.run(window, 5)).reshape(n, qh, dim)
    assert not np.isfinite(got[n - 2:]).any()
    if kind == "mxfp4":
        c.cache.v_scale[page, :, off] = 127
    else:
        c.cache.v[page, :, off] = 1.0
    k, v = held(c.cache)
    want, mag, prod, seen = oracle.attention(f64(c.q).reshape(n, qh, dim), k, v, c.offs, c.kv_lens, c.table, 16, qh,
                                             window, 5, 1 / math.sqrt(dim), c.pages)
    bound = oracle.attention_bound(want, mag, prod, seen, dim, qt, 24 if qt is F32 else 8)
    assert (np.abs(got - want) <= bound)[:n - 2].all()


@pytest.mark.parametrize("qt,kind", [(F32, "bf16"), (F32, "mxfp4"), (BF16, "bf16"), (BF16, "mxfp4")])
@pytest.mark.parametrize("n,kv", [(4, 40), (3, 1500)])
def test_unseen_values_of_few_rows(gpu_device, qt, kind, n, kv):
    note(f"unseen by few rows {qt} {kind} {n} {kv}")
    c = Case(gpu_device, qt, kind, 2, 2, 64, 16, [n], [kv], seed=4)
    page, off = c.table[0, (kv - 2) // 16], (kv - 2) % 16
    if kind == "mxfp4":
        c.cache.v_scale[page, :, off] = 255
    else:
        c.cache.v[page, :, off] = float("inf")
    got = f64(c.run(1 << 30, 0)).reshape(n, -1)
    assert np.isfinite(got[:n - 2]).all() and not np.isfinite(got[n - 2:]).any()


@pytest.mark.parametrize("qt,kind", [(F32, "f32"), (F32, "bf16"), (F32, "mxfp4"), (BF16, "bf16"), (BF16, "mxfp4")])
@pytest.mark.parametrize("q_lens,kv_lens", [([4, 20], [60, 20]), ([100], [130])])
def test_unseen_values_do_not_reach_a_row(gpu_device, qt, kind, q_lens, kv_lens):
    """NaN and infinite keys and values that a later or windowed row sees, and
    this one does not."""
    note(f"unseen {qt} {kind} {q_lens}")
    c = Case(gpu_device, qt, kind, 8, 2, 64, 16, q_lens, kv_lens, seed=8)
    window, sinks = 9, 2
    bad = {}
    for b, n in enumerate(kv_lens):
        for j, which in ((n - 1, "v"), (n - 3, "k"), (n - q_lens[b] - 1, "v")):
            if j < 0:
                continue
            page, off = c.table[b, j // 16], j % 16
            if kind == "mxfp4":
                getattr(c.cache, which + "_scale")[page, :, off] = 255
            else:
                getattr(c.cache, which)[page, :, off] = float("inf") if which == "v" else float("nan")
            bad[(b, j)] = which
    got = f64(c.run(window, sinks)).reshape(c.rows, -1)
    hit = np.zeros(c.rows, bool)
    for b, n in enumerate(kv_lens):
        for i in range(q_lens[b]):
            p = n - q_lens[b] + i
            hit[c.offs[b] + i] = any(bb == b and j <= p and (j > p - window or j < sinks) for bb, j in bad)
    assert hit.any() and not hit.all()
    assert np.isfinite(got[~hit]).all()
    assert not np.isfinite(got[hit]).all(axis=1).any()
    # the clean rows are those of the same batch without the bad entries
    for (b, j), which in bad.items():
        page, off = c.table[b, j // 16], j % 16
        if kind == "mxfp4":
            getattr(c.cache, which + "_scale")[page, :, off] = 127
        else:
            getattr(c.cache, which)[page, :, off] = 1.0
    k, v = held(c.cache)
    want, mag, prod, seen = oracle.attention(f64(c.q).reshape(c.rows, 8, 64), k, v, c.offs, c.kv_lens, c.table, 16, 8,
                                             window, sinks, 1 / 8, c.pages)
    bound = oracle.attention_bound(want, mag, prod, seen, 64, qt, 24 if qt is F32 else 8).reshape(c.rows, -1)
    assert (np.abs(got - want.reshape(c.rows, -1)) <= bound)[~hit].all()


@pytest.mark.parametrize("qt,kind", [(F32, "f32"), (F32, "bf16"), (F32, "mxfp4"), (BF16, "bf16"), (BF16, "mxfp4")])
@pytest.mark.parametrize("qh,kvh,n,kv,window,back", [(32, 1, 4, 60, 2047, 0),    # 32 rows a token
                                                     (32, 1, 4, 60, 3, 4), (64, 1, 2, 1500, 2047, 0),
                                                     (8, 2, 41, 97, 3, 8)])       # one token behind full ones
def test_unseen_values_of_other_tokens(gpu_device, qt, kind, qh, kvh, n, kv, window, back):
    """A value that is not finite, `back` keys before the last, and groups of
    rows that are one token's, whose neighbours' keys it does not see."""
    note(f"other tokens {qt} {kind} {qh}/{kvh} {n} {kv} {window}")
    c = Case(gpu_device, qt, kind, qh, kvh, 64, 16, [n], [kv], seed=5)
    j = kv - 1 - back
    page, off = c.table[0, j // 16], j % 16
    if kind == "mxfp4":
        c.cache.v_scale[page, :, off] = 255
    else:
        c.cache.v[page, :, off] = float("inf")
    got = f64(c.run(window, 0)).reshape(n, -1)
    at = np.arange(kv - n, kv)
    hit = (j <= at) & (j > at - window)
    assert hit.any() and not hit.all()
    assert np.isfinite(got[~hit]).all() and not np.isfinite(got[hit]).any()


@pytest.mark.parametrize("qt,kind", [(F32, "bf16"), (BF16, "mxfp4")])
def test_rows_left_alone_and_pages_left_out(gpu_device, qt, kind):
    """Rows behind the last sequence and past max_q_len keep their bytes; page
    ids outside the cache leave their keys out; slices of wider rows."""
    note(f"rows left alone {qt} {kind}")
    for q_lens, kv_lens in (([2, 3], [40, 70]), ([80, 30], [100, 50])):
        c = Case(gpu_device, qt, kind, 8, 2, 128, 16, q_lens, kv_lens, extra_rows=4, seed=5)
        c.table[1, 1], c.table[0, 0] = c.pages + 3, -7
        out = torch.full((c.rows, 8 * 128), 7.0, dtype=qt, device=gpu_device)
        wide = torch.zeros(c.rows, 8 * 128 + 64, dtype=qt, device=gpu_device)
        wide[:, 64:] = c.q
        c.q = wide[:, 64:]
        got = c.run(2047, 1, out=out)
        assert got is out and bool((out[sum(q_lens):] == 7.0).all())
        c.check(got, 2047, 1)
        short = torch.full_like(out, 5.0)
        c.run(2047, 1, out=short, max_q_len=2)
        keep = torch.from_numpy(np.concatenate([[True, True] + [False] * (n - 2) for n in q_lens] + [[False] * 4]))
        keep = keep.to(gpu_device)
        assert bool((short[~keep] == 5.0).all())
        # fewer queries may take another kernel: its rows are held to the same bound
        c.check(torch.where(keep[:, None], short, out), 2047, 1)


@pytest.mark.parametrize("qt,kind", [(F32, "f32"), (F32, "mxfp4"), (BF16, "bf16")])
def test_pages_that_sequences_share(gpu_device, qt, kind):
    """A common prefix held once: sequences whose tables name the same pages,
    one of them twice the same sequence, and slots read back more than once."""
    note(f"shared pages {qt} {kind}")
    c = Case(gpu_device, qt, kind, 8, 2, 64, 16, [1, 40, 1, 2], [70, 70, 70, 66], seed=6)
    c.table[1:] = c.table[0]
    c.check(c.run(1 << 30, 0), 1 << 30, 0)
    c.check(c.run(20, 3), 20, 3)
    slots = torch.tensor([int(c.table[0, 1]) * 16 + 3] * 5, device=c.dev)
    for t in serve.kv_gather_gpu(c.cache, slots):
        assert torch.equal(t, t[:1].expand_as(t)) and t.isfinite().all()


@pytest.mark.parametrize("qt,kind", [(F32, "f32"), (F32, "bf16"), (BF16, "mxfp4")])
def test_table_entries_that_no_query_sees(gpu_device, qt, kind):
    """Entries past the length and before the window hold anything."""
    note(f"unseen entries {qt} {kind}")
    for q_lens, kv_lens in (([1, 2], [150, 90]), ([50, 3], [170, 40])):
        c = Case(gpu_device, qt, kind, 8, 2, 64, 16, q_lens, kv_lens, seed=9)
        want = c.run(30, 2)
        wide = np.full((2, c.table.shape[1] + 5), 0x7FFFFFFF, np.int32)
        wide[:, :c.table.shape[1]] = c.table
        for b, n in enumerate(kv_lens):
            first = max((n - q_lens[b] + 1 - 30) // 16, 1)
            wide[b, 1:first] = -0x80000000
            wide[b, -(-n // 16):] = 0x7FFFFFFF
        c.table = wide
        assert torch.equal(bits(c.run(30, 2)), bits(want))


def test_lengths_past_the_bounds_are_cut(gpu_device):
    """kv_lens past max_kv_len or the table, offsets past the rows: nothing is
    read or written outside the arrays."""
    c = Case(gpu_device, BF16, "bf16", 4, 1, 64, 16, [1, 2], [30, 48], seed=2)
    c.kv_lens[:] = [1 << 30, 1 << 20]
    c.max_kv = 1 << 30
    a = c.run(64, 0)                     # cut to the table: 48 positions each
    assert a.shape == (3, 256)
    c.kv_lens[:] = [48, 48]
    c.max_kv = 48
    b = c.run(64, 0)
    assert torch.equal(a[1:], b[1:])     # row 0's second pages are the -1 of the table: left out on both
    c.offs[:] = [-5, 1, 1 << 20]
    assert c.run(64, 0, max_q_len=3).shape == (3, 256)


def test_scale_and_large_scores(gpu_device):
    for scale in (0.0, -0.5, 3.0):
        c = Case(gpu_device, F32, "bf16", 4, 2, 64, 16, [2, 1], [40, 70], seed=4)
        c.check(c.run(50, 3, scale=scale), 50, 3, scale=scale)
    c = Case(gpu_device, F32, "f32", 4, 2, 64, 16, [2, 1], [40, 70], seed=4)
    c.q *= 100.0                          # one key takes all the weight
    got = c.run(50, 3)
    assert bool(torch.isfinite(got).all())


def test_offsets_past_32_bits(gpu_device):
    """Pages behind the first 2^32 elements (and bytes) of a cache."""
    dev, page, kvh, dim = gpu_device, 256, 4, 128
    pages = (1 << 32) // (kvh * page * dim) + 8
    small = Case(dev, BF16, "bf16", 16, kvh, dim, page, [3, 1], [300, 600], seed=6)
    k, v = (torch.empty(pages, kvh, page, dim, dtype=BF16, device=dev) for _ in range(2))
    k[-small.pages:], v[-small.pages:] = small.cache.k, small.cache.v
    want = small.run(400, 4)
    small.cache = serve.PagedKvCache(k, v)
    small.table = np.where(small.table >= 0, small.table + pages - small.pages, -1).astype(np.int32)
    assert torch.equal(small.run(400, 4), want)
    slots = torch.tensor([pages * page - 1, (pages - 1) * page], device=dev)
    x = torch.randn(2, kvh * dim, dtype=BF16, device=dev)
    pos = torch.zeros(2, dtype=torch.int32, device=dev)
    cos, sin = torch.ones(1, dim // 2, device=dev), torch.zeros(1, dim // 2, device=dev)
    serve.kv_append_gpu(small.cache, x, x, pos, slots, cos, sin)
    for got in serve.kv_gather_gpu(small.cache, slots, BF16):
        assert torch.equal(got, x)


@pytest.mark.parametrize("qt,kind", [(F32, "bf16"), (BF16, "bf16"), (BF16, "mxfp4"), (F32, "f32")])
def test_step_in_a_graph_and_on_another_stream(gpu_device, qt, kind):
    """append + attention recorded once and replayed while lengths, slots and
    values change, with eager work between; and run on a side stream."""
    dev = gpu_device
    note(f"graph {qt} {kind}")
    rng = np.random.default_rng(1)
    kvh, qh, dim, page, batch = 2, 8, 128, 16, 3
    cache = make_cache(kind, 3 * 80, kvh, page, dim, dev, rng)
    table = torch.arange(3 * 80, dtype=torch.int32, device=dev).view(batch, 80)
    cos, sin = (torch.from_numpy(a).to(dev) for a in attention.rope_table(1280, dim))
    offs = torch.arange(batch + 1, dtype=torch.int32, device=dev)
    lens = torch.zeros(batch, dtype=torch.int32, device=dev)
    pos, slots = torch.zeros_like(lens), torch.zeros(batch, dtype=torch.int64, device=dev)
    row = torch.zeros(batch, (qh + 2 * kvh) * dim, dtype=qt, device=dev)

    def step(out=None):
        q, k, v = row.split([qh * dim, kvh * dim, kvh * dim], 1)
        q = serve.kv_append_gpu(cache, k, v, pos, slots, cos, sin, q=q)
        return serve.attention_paged_gpu(q, cache, offs, lens, table, 1, 1280, q_heads=qh, window=1 << 30, out=out)

    def feed(n):
        g = torch.Generator(dev).manual_seed(n)
        row.copy_(torch.randn(row.shape, generator=g, device=dev).to(qt))
        lens.copy_(torch.tensor([n, n + 500, 2 * n], dtype=torch.int32))
        pos.copy_(lens - 1)
        slots.copy_(table.gather(1, (pos // page)[:, None].long())[:, 0].long() * page + pos % page)

    feed(10)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in (1, 17, 300, 17, 600):
        feed(n)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(bits(got), bits(want)), n
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream(dev))
            other = step()
        side.synchronize()
        assert torch.equal(bits(other), bits(want)), n


@pytest.mark.parametrize("qt,kind", [(F32, "bf16"), (BF16, "mxfp4"), (F32, "f32")])
@pytest.mark.parametrize("q_lens,kv_lens", [([1] * 70 + [2], [7 + 3 * i for i in range(71)]),
                                            ([11] * 66, [20 + 2 * i for i in range(66)]),
                                            ([1, 40] * 35, [50 + i for i in range(70)])])
def test_many_sequences(gpu_device, qt, kind, q_lens, kv_lens):
    """More sequences than a wave has lanes."""
    note(f"many sequences {qt} {kind} {len(q_lens)}")
    c = Case(gpu_device, qt, kind, 4, 1, 64, 16, q_lens, kv_lens, seed=12)
    c.check(c.run(40, 2), 40, 2)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 2], [1800, 1500]), ([40], [1700]), ([50, 1], [1300, 1900])])
def test_split_rows_left_alone(gpu_device, q_lens, kv_lens):
    """The join of a split key axis writes the rows of the sequences alone."""
    for qt, kind in ((BF16, "bf16"), (F32, "mxfp4")):
        note(f"split rows left alone {qt} {kind} {q_lens}")
        c = Case(gpu_device, qt, kind, 4, 1, 128, 16, q_lens, kv_lens, extra_rows=5, seed=9)
        c.offs[:] = c.offs + 2                       # two rows before the first sequence, three behind the last
        out = torch.full((c.rows, 4 * 128), 3.0, dtype=qt, device=gpu_device)
        c.run(1 << 30, 0, out=out)
        n = sum(q_lens)
        assert bool((out[:2] == 3.0).all()) and bool((out[2 + n:] == 3.0).all())
        c.q, c.offs, c.rows = c.q[2:2 + n].contiguous(), c.offs - 2, n
        c.check(out[2:2 + n], 1 << 30, 0)


@pytest.mark.parametrize("qt,kind", [(F32, "f32"), (F32, "bf16"), (BF16, "mxfp4")])
@pytest.mark.parametrize("q_lens,kv_lens", [([3, 1], [40, 50]), ([60, 2], [90, 64])])
def test_a_row_that_is_nan_stays_alone(gpu_device, qt, kind, q_lens, kv_lens):
    c = Case(gpu_device, qt, kind, 4, 2, 64, 16, q_lens, kv_lens, seed=21)
    clean = f64(c.run(64, 1))
    c.q[1] = float("nan")
    got = f64(c.run(64, 1))
    assert np.isnan(got[1]).all()
    keep = np.arange(c.rows) != 1
    assert np.array_equal(got[keep], clean[keep])


def test_two_graphs_at_once(gpu_device):
    """Two recorded calls replayed together on two streams share nothing."""
    dev = gpu_device
    cases = [Case(dev, BF16, "bf16", 8, 2, 128, 16, [1, 1], [1900, 1500], seed=31),
             Case(dev, F32, "mxfp4", 8, 2, 128, 16, [2, 40], [1200, 300], seed=32)]
    side = [torch.cuda.Stream(dev), torch.cuda.Stream(dev)]
    graphs, outs, want = [], [], []
    for c in cases:
        args = (c.up(c.offs), c.up(c.kv_lens), c.up(c.table), c.max_q, c.max_kv)
        call = lambda c=c, args=args: serve.attention_paged_gpu(c.q, c.cache, *args, q_heads=8, window=1 << 30)  # noqa: E731
        want.append(call().clone())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append((g, args))
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for (g, _a), st in zip(graphs, side):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(bits(o), bits(w))


def test_attention_of_nothing(gpu_device):
    c = Case(gpu_device, BF16, "bf16", 4, 1, 64, 16, [1, 1], [5, 7], seed=2)
    e = torch.empty(0, dtype=torch.int32, device=gpu_device)
    got = serve.attention_paged_gpu(c.q[:0], c.cache, torch.zeros(1, dtype=torch.int32, device=gpu_device), e,
                                    torch.empty(0, 1, dtype=torch.int32, device=gpu_device), 0, 0, q_heads=4,
                                    window=8)
    assert got.shape == (0, 256)
    c.kv_lens[:] = 0
    assert bool((c.run(8, 2, max_kv_len=0) == 0).all())


# ---- the logits' rules -------------------------------------------------------------

def _logit_case(dev, dtype, rows, vocab, hist, bias, mask, seed):
    rng = np.random.default_rng(seed)
    x = (4 * rng.standard_normal((rows, vocab))).astype(np.float32)
    x[:, vocab // 2] = 0.0
    x[0, 0] = -0.0
    x = torch.from_numpy(x).to(dtype)
    h = np.floor(vocab * rng.random((rows, hist)) ** 3).astype(np.int32)
    if hist > 3:
        h[:, 0], h[:, 1], h[:, 2] = -1, vocab, 1 << 30        # no tokens of this vocabulary
    lens = rng.integers(0, hist + 1, rows).astype(np.int32)
    lens[0] = hist + 9                                        # cut to the list
    r = dict(history=h, history_lens=lens, prompt_lens=(lens // 3).astype(np.int32),
             repetition=(1 + rng.random(rows)).astype(np.float32), frequency=rng.random(rows).astype(np.float32),
             presence=rng.random(rows).astype(np.float32))
    if bias:
        r["bias_ids"] = rng.integers(-1, vocab + 1, (rows, bias)).astype(np.int32)
        r["bias_ids"][:, -1] = r["bias_ids"][:, 0]            # named twice: the last counts
        r["bias_values"] = rng.standard_normal((rows, bias)).astype(np.float32)
        r["bias_lens"] = np.full(rows, bias, np.int32)
        r["bias_lens"][-1] = bias // 2
    if mask:
        r["mask"] = rng.integers(-2 ** 31, 2 ** 31, (4, (vocab + 31) // 32 + 1)).astype(np.int32)
        r["mask"][3] = 0                                      # nothing is allowed
        r["mask_index"] = rng.integers(-1, 6, rows).astype(np.int32)
        r["mask_index"][0] = 3
    return x.to(dev), r


def _logit_want(x, r):
    rows, vocab = x.shape
    out = []
    for i in range(rows):
        n = min(int(r["history_lens"][i]), r["history"].shape[1])
        bias = {}
        if "bias_ids" in r:
            for t, b in list(zip(r["bias_ids"][i], r["bias_values"][i]))[:r["bias_lens"][i]]:
                bias[int(t)] = b
        allowed = None
        if "mask" in r and 0 <= r["mask_index"][i] < 4:
            w = r["mask"][r["mask_index"][i]].view(np.uint32)
            allowed = (w[np.arange(vocab) // 32] >> (np.arange(vocab) % 32) & 1).astype(bool)
        out.append(oracle.logits(x[i].float().cpu().numpy(), i, r["history"][i, :n].tolist(), int(r["prompt_lens"][i]),
                                 r["repetition"][i], r["frequency"][i], r["presence"][i], bias, allowed))
    return torch.from_numpy(np.stack(out)).to(x.dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,hist,bias,mask", [
    (1, 1, 1, 0, False), (3, 33, 8, 4, True), (2, 4096, 100, 0, True), (5, 4097, 700, 300, False),
    (2, 32064, 613, 10, True), (7, 1003, 0, 5, True), (1, 8191, 2000, 1, True)])
def test_logits(gpu_device, dtype, rows, vocab, hist, bias, mask):
    note(f"logits {dtype} {rows} x {vocab} history {hist} bias {bias} mask {mask}")
    x, r = _logit_case(gpu_device, dtype, rows, vocab, hist, bias, mask, seed=vocab)
    t = {n: torch.from_numpy(a).to(gpu_device) for n, a in r.items()}
    want = _logit_want(x, r)
    assert torch.equal(bits(serve.logits_process_gpu(x, **t)), bits(want))
    # a slice of a wider row whose start is off the vectors' alignment, in place
    wide = torch.full((rows, vocab + 3), 9.0, dtype=dtype, device=gpu_device)
    wide[:, 1:vocab + 1] = x
    inner = wide[:, 1:vocab + 1]
    got = serve.logits_process_gpu(inner, out=inner, **t)
    assert got.data_ptr() == inner.data_ptr() and torch.equal(bits(inner), bits(want))
    assert bool((wide[:, 0] == 9.0).all()) and bool((wide[:, vocab + 1:] == 9.0).all())


@pytest.mark.parametrize("rows,vocab", [(64, 2049), (67, 1030), (131, 6100)])
def test_logits_of_many_rows(gpu_device, rows, vocab):
    """Rows dealt to the XCDs, their number no multiple of 8 among them."""
    test_logits(gpu_device, BF16, rows, vocab, 60, 3, True)


def test_logits_rules_alone(gpu_device):
    """Each rule without the others; no rule at all copies the logits."""
    x, r = _logit_case(gpu_device, F32, 4, 777, 50, 6, True, seed=11)
    t = {n: torch.from_numpy(a).to(gpu_device) for n, a in r.items()}
    assert torch.equal(bits(serve.logits_process_gpu(x)), bits(x))
    only_hist = {n: t[n] for n in ("history", "history_lens")}
    assert torch.equal(bits(serve.logits_process_gpu(x, **only_hist)), bits(x))
    one, zero = np.ones(4, np.float32), np.zeros(4, np.float32)
    for name in ("repetition", "frequency", "presence"):
        q = {**r, "repetition": one, "frequency": zero, "presence": zero, name: r[name]}
        for other in ("bias_ids", "bias_values", "bias_lens", "mask", "mask_index"):
            q.pop(other)
        got = serve.logits_process_gpu(x, prompt_lens=t["prompt_lens"], **only_hist, **{name: t[name]})
        assert torch.equal(bits(got), bits(_logit_want(x, q)))
    got = serve.logits_process_gpu(x, mask=t["mask"])          # row r has mask r
    q = {**r, "history_lens": np.zeros(4, np.int32), "mask_index": np.arange(4, dtype=np.int32)}
    for other in ("bias_ids", "bias_values", "bias_lens"):
        q.pop(other)
    assert torch.equal(bits(got), bits(_logit_want(x, q)))


def test_logits_in_a_graph_and_on_another_stream(gpu_device):
    dev = gpu_device
    x, r = _logit_case(dev, F32, 3, 5000, 90, 7, True, seed=2)
    t = {n: torch.from_numpy(a).to(dev) for n, a in r.items()}
    want = bits(_logit_want(x, r))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = serve.logits_process_gpu(x, **t)
    side.synchronize()
    assert torch.equal(bits(got), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = serve.logits_process_gpu(x, **t)
    for _ in range(4):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(out), want)
        serve.logits_process_gpu(x)
        t["history_lens"].add_(0)
    t["history_lens"].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(bits(out), bits(_logit_want(x, {**r, "history_lens": np.zeros(3, np.int32)})))


def test_logits_that_are_not_finite(gpu_device):
    """NaN stays NaN where the mask allows it, and is -inf where it does not."""
    x = torch.tensor([[float("nan"), float("inf"), -float("inf"), 1.0]], device=gpu_device)
    mask = torch.tensor([[0b1011]], dtype=torch.int32, device=gpu_device)
    got = serve.logits_process_gpu(x, mask=mask).cpu()[0].tolist()
    assert math.isnan(got[0]) and got[1:] == [math.inf, -math.inf, 1.0]
    mask[0, 0] = 0b1000
    assert serve.logits_process_gpu(x, mask=mask).cpu()[0].tolist() == [-math.inf] * 3 + [1.0]
