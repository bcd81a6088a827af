"""The quantized key / value cache: written, read back, attended to, against 64 bits."""
import numpy as np
import pytest
import torch

from iconnx_amd import ops
from tests import decoder_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
TERMS = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}


def some(shape, dtype, seed, spread=6):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-spread, spread + 1, shape[:-1] + (1,), generator=g).float())
    x[..., ::13] *= 5.0
    return x.to(dtype).cuda()


def same(t, want, dtype):
    want = torch.from_numpy(want).to(dtype).double()
    assert torch.equal(torch.nan_to_num(t.double().cpu(), nan=12345.0), torch.nan_to_num(want, nan=12345.0))


# ---- writing and reading -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("H,D,page,T", [(1, 32, 16, 1), (3, 64, 16, 50), (2, 96, 48, 33), (8, 128, 16, 100), (1, 160, 32, 40),
                                        (2, 224, 16, 20), (4, 256, 128, 70)])
def test_write_then_read(H, D, page, T, bits, dtype):
    pages = -(-T // page) + 2
    cache = ops.KvCache(pages, page, H, D, bits=bits)
    k, v = some((T, H, D), dtype, T), some((T, H, D), dtype, T + 1)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(D))[:T].cuda()
    ops.gpu_kv_cache_write(cache, k, v, slots)
    rk, rv = ops.gpu_kv_cache_read(cache, slots.int(), dtype=dtype)
    same(rk, ref.cached(k, bits), dtype)
    same(rv, ref.cached(v, bits), dtype)
    # the slots that were not written still hold zeros
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots] = False
    for t in ops.gpu_kv_cache_read(cache, torch.nonzero(rest).flatten()):
        assert not t.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("T,first", [(16, 0), (64, 16), (100, 3), (37, 30), (257, 16)])
def test_runs_of_consecutive_slots(T, first, bits, dtype):
    """Prompts: consecutive tokens into consecutive slots, from the start of a chunk and from inside one."""
    H, D, page = 3, 128, 64
    cache = ops.KvCache(6, page, H, D, bits=bits)
    k, v = some((T, H, D), dtype, T), some((T, H, D), dtype, T + 1)
    slots = torch.arange(first, first + T).cuda()
    ops.gpu_kv_cache_write(cache, k, v, slots)
    rk, rv = ops.gpu_kv_cache_read(cache, slots, dtype=dtype)
    same(rk, ref.cached(k, bits), dtype)
    same(rv, ref.cached(v, bits), dtype)
    back = slots.flip(0)
    rk, rv = ops.gpu_kv_cache_read(cache, back, dtype=torch.float32)
    same(rk.flip(0), ref.cached(k, bits), torch.float32)
    same(rv.flip(0), ref.cached(v, bits), torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("H,D,page,T", [(256, 32, 32, 130), (256, 64, 16, 131), (128, 96, 64, 257), (64, 128, 16, 520), (64, 160, 48, 515),
                                        (32, 192, 16, 1030), (32, 224, 32, 1025), (32, 256, 128, 1041)])
def test_many_tokens(H, D, page, T, bits, dtype):
    """Prompts of several sequences, which start at and inside chunks of 16 in shuffled pages, a few tokens passed
    over, and some alone in their pages."""
    pages = -(-T // page) + 9
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(T))
    at = torch.arange(T)
    slots = order[at // page] * page + at % page
    cut = T // 3 + 5  # the rest starts inside a page, out of step with the chunks
    slots[cut:] = (at[cut:] - cut + 3) % page + order[3 + (at[cut:] - cut + 3) // page + cut // page] * page
    slots[-3:] = order[-3:] * page + torch.tensor([0, 7, 15])
    slots[cut + 40:cut + 43] = -1
    k, v = some((T, H, D), dtype, T), some((T, H, D), dtype, T + 1)
    big, small = ops.KvCache(pages, page, H, D, bits=bits), ops.KvCache(pages, page, H, D, bits=bits)
    ops.gpu_kv_cache_write(big, k, v, slots.cuda())
    for i in range(0, T, 16):  # the same in pieces
        ops.gpu_kv_cache_write(small, k[i:i + 16], v[i:i + 16], slots[i:i + 16].cuda())
    assert torch.equal(big.data, small.data)
    rk, rv = ops.gpu_kv_cache_read(big, slots.cuda(), dtype=dtype)
    parts = [ops.gpu_kv_cache_read(big, slots[i:i + 16].cuda(), dtype=dtype) for i in range(0, T, 16)]
    assert torch.equal(rk, torch.cat([x[0] for x in parts])) and torch.equal(rv, torch.cat([x[1] for x in parts]))
    rows, heads = torch.cat([torch.arange(0, 20), torch.arange(cut - 2, cut + 50), torch.arange(T - 8, T)]), torch.arange(3, H, 11)
    gone = (slots[rows] < 0).numpy()
    for got, x in ((rk, k), (rv, v)):
        want = ref.cached(x[rows.cuda()][:, heads.cuda()], bits)
        want[gone] = 0
        same(got[rows.cuda()][:, heads.cuda()], want, dtype)


@pytest.mark.parametrize("bits", [4, 8])
def test_every_code_tie_and_scale_limit(bits):
    grid = ref.GRID[bits]
    ties = (grid[1:] + grid[:-1]) / 2
    values = np.concatenate([grid, ties, np.nextafter(ties, 0), np.nextafter(ties, 1e9)]).astype(np.float32)
    values = np.concatenate([values, -values])
    rows = []
    for top in ((6.0, 6.9, 7.0, 7.5) if bits == 4 else (448.0, 463.9, 464.0, 464.1, 479.0)):
        for e in (-130, -118, -100, -3, 0, 60, 119, 125):
            for i in range(0, len(values), 31):
                r = np.zeros(32, np.float64)
                part = values[i:i + 31]
                part = part[np.abs(part) <= top]
                r[1:1 + len(part)] = part
                r[0] = top
                r *= 2.0 ** e
                rows.append(np.where(np.abs(r) > 3.4028e38, 3.4028e38 * np.sign(r), r))
    x = torch.from_numpy(np.array(rows)).float().view(-1, 1, 32).cuda()
    cache = ops.KvCache(-(-len(x) // 16), 16, 1, 32, bits=bits)
    slots = torch.arange(len(x)).cuda()
    ops.gpu_kv_cache_write(cache, x, x.flip(2), slots)
    k, v = ops.gpu_kv_cache_read(cache, slots)
    same(k, ref.cached(x, bits), torch.float32)
    same(v, ref.cached(x.flip(2), bits), torch.float32)


@pytest.mark.parametrize("bits", [4, 8])
def test_blocks_that_are_not_finite_read_back_as_nan(bits):
    x = torch.randn(20, 2, 64).cuda()
    x[3, 0, 5] = float("nan")
    x[9, 1, 63] = float("inf")
    x[17, 0, 33] = -float("inf")
    cache = ops.KvCache(2, 16, 2, 64, bits=bits)
    slots = torch.arange(20).cuda()
    ops.gpu_kv_cache_write(cache, x, x, slots)
    for t in ops.gpu_kv_cache_read(cache, slots):
        same(t, ref.cached(x, bits), torch.float32)


@pytest.mark.parametrize("bits", [4, 8])
def test_slots_outside_the_cache_are_passed_over(bits):
    cache = ops.KvCache(2, 16, 2, 64, bits=bits)
    x = some((40, 2, 64), torch.float32, 1)
    slots = torch.arange(40).cuda()
    slots[7], slots[12] = -1, -(1 << 40)
    slots[20] = 1 << 33
    ops.gpu_kv_cache_write(cache, x, x, slots)  # 32 .. 39 are past the end too
    inside = ((slots >= 0) & (slots < 32)).cpu().numpy()
    want = ref.cached(x, bits)
    want[~inside] = 0
    for t in ops.gpu_kv_cache_read(cache, slots):
        same(t, want, torch.float32)
    untouched = ops.gpu_kv_cache_read(cache, torch.tensor([7, 12, 20]).cuda())
    assert not untouched[0].any() and not untouched[1].any()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,odd", [(64, 0), (96, 1), (128, 3)])
def test_slices_of_a_fused_projection(dtype, bits, D, odd):
    T, H = 70, 3
    flat = some((T, 3 * H * D + odd), dtype, 4, spread=2)
    part = flat[:, odd:].unflatten(1, (3, H, D))  # rows that start at odd elements
    cache, dense = ops.KvCache(8, 16, H, D, bits=bits), ops.KvCache(8, 16, H, D, bits=bits)
    slots = torch.arange(5, 5 + T).cuda()
    ops.gpu_kv_cache_write(cache, part[:, 1], part[:, 2], slots)
    ops.gpu_kv_cache_write(dense, part[:, 1].contiguous(), part[:, 2].contiguous(), slots)
    assert torch.equal(cache.data, dense.data)
    same(ops.gpu_kv_cache_read(cache, slots, dtype=dtype)[1], ref.cached(part[:, 2], bits), dtype)


def test_no_tokens():
    cache = ops.KvCache(1, 16, 1, 32)
    none = torch.empty(0, 1, 32).cuda()
    ops.gpu_kv_cache_write(cache, none, none, torch.empty(0, dtype=torch.int64).cuda())
    k, v = ops.gpu_kv_cache_read(cache, torch.empty(0, dtype=torch.int32).cuda(), dtype=torch.bfloat16)
    assert k.shape == v.shape == (0, 1, 32)


# ---- attention ---------------------------------------------------------------------------------
class Filled:
    """A cache of `lengths` tokens a sequence in shuffled pages, every other slot holding what must not matter."""

    def __init__(self, lengths, Hkv, D, page, bits, seed=0, spare=0, garbage=True):
        self.lengths, self.D, self.page, self.bits = lengths, D, page, bits
        width = max([1] + [-(-n // page) for n in lengths]) + spare
        pages = len(lengths) * width + 2
        self.cache = ops.KvCache(pages, page, Hkv, D, bits=bits)
        g = torch.Generator().manual_seed(seed)
        self.table = torch.randperm(pages, generator=g)[: len(lengths) * width].view(len(lengths), width).int()
        if garbage:
            x = torch.full((pages * page, Hkv, D), float("nan")).cuda()
            ops.gpu_kv_cache_write(self.cache, x, x, torch.arange(pages * page).cuda())
        self.k, self.v = [], []
        for b, n in enumerate(lengths):
            k, v = torch.randn(n, Hkv, D, generator=g) * 1.5, torch.randn(n, Hkv, D, generator=g)
            self.put(b, k, v)
            self.k.append(ref.cached(k, bits))
            self.v.append(ref.cached(v, bits))

    def slots(self, b, n):
        j = torch.arange(n)
        return self.table[b][j // self.page].long() * self.page + j % self.page

    def put(self, b, k, v):
        if len(k):
            ops.gpu_kv_cache_write(self.cache, k.cuda(), v.cuda(), self.slots(b, len(k)).cuda())

    def attend(self, q, rows=None, **kw):
        starts = None if rows is None else torch.tensor(np.cumsum([0] + list(rows)), dtype=torch.int32).cuda()
        return ops.gpu_kv_cache_attention(q, self.cache, self.table.cuda(), torch.tensor(self.lengths, dtype=torch.int32).cuda(),
                                          q_starts=starts, **kw)

    def check(self, q, rows=None, **kw):
        out = self.attend(q, rows, **kw)
        assert out.dtype == q.dtype and out.shape == q.shape
        kw.pop("max_rows", None)
        kw.pop("out", None)
        sl = kw.pop("slopes", None)
        starts = np.cumsum([0] + ([1] * len(self.lengths) if rows is None else list(rows)))
        want, bound = ref.attention(q, self.k, self.v, self.lengths, starts, kw.pop("scale", self.D ** -0.5),
                                    slopes=None if sl is None else ref.f64(sl), terms=TERMS[q.dtype], dtype=q.dtype, **kw)
        n = starts[-1]
        err = np.abs(ref.f64(out[:n]) - want[:n])
        worst = np.unravel_index((err / bound[:n]).argmax(), err.shape) if n else 0
        assert not np.isnan(err).any() and (err <= bound[:n]).all(), "off by %g where %g is allowed, at %s" % (err[worst], bound[worst], worst)
        return out


def query(rows, H, D, dtype, seed=7):
    return torch.randn(rows, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(1, 1, 32, 16), (12, 12, 64, 16), (6, 2, 96, 32), (8, 2, 128, 16), (5, 1, 160, 48),
                                           (16, 1, 192, 16), (7, 1, 256, 64), (40, 2, 64, 16)])
def test_one_token_a_sequence(Hq, Hkv, D, page, bits, dtype):
    f = Filled([1, 16, 17, 31, 33, 100, 257, 0], Hkv, D, page, bits)
    f.check(query(8, Hq, D, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(2, 2, 64, 16), (4, 1, 128, 32), (3, 1, 96, 16), (6, 2, 256, 16)])
def test_chunks_of_rows(Hq, Hkv, D, page, bits, dtype):
    rows = [1, 5, 40, 33, 0, 70, 3]
    f = Filled([90, 5, 40, 100, 20, 130, 64], Hkv, D, page, bits)
    f.check(query(sum(rows), Hq, D, dtype), rows)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("Hq,Hkv,D,rows", [(2, 2, 64, [33, 64, 17, 1]), (6, 2, 96, [21, 16, 0, 11]), (4, 1, 256, [16, 13, 1, 5])])
def test_up_to_four_tiles_of_rows(Hq, Hkv, D, rows, bits, dtype):
    f = Filled([90, 64, 600, 11], Hkv, D, 16, bits)
    f.check(query(sum(rows), Hq, D, dtype), rows, max_rows=max(rows))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=20), dict(window=1000), dict(softcap=3.0), dict(softcap=30.0, window=50),
                                dict(slopes=True), dict(slopes=True, softcap=10.0, window=33), dict(causal=False),
                                dict(causal=False, window=40, slopes=True), dict(scale=0.5), dict(scale=-0.2), dict(scale=0.0)])
def test_masks_and_scores(kw, dtype):
    kw = dict(kw)
    rows = [1, 37, 64, 2]
    f = Filled([150, 37, 200, 65], 2, 64, 16, 4, spare=2)
    if kw.get("slopes"):
        kw["slopes"] = torch.exp2(-torch.arange(1, 5).float()).cuda()
    f.check(query(sum(rows), 4, 64, dtype), rows, **kw)
    f.check(query(4, 4, 64, dtype), **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,rows", [([3000], None), ([5000, 10, 0, 2049], None), ([1500], [130]), ([2100, 700], [1, 300])])
def test_long_sequences(lengths, rows, dtype):
    """Tokens in shares that are joined."""
    f = Filled(lengths, 1, 64, 16, 4)
    n = len(lengths) if rows is None else sum(rows)
    f.check(query(n, 4, 64, dtype), rows)
    f.check(query(n, 4, 64, dtype), rows, window=777)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [None, [3, 50]])
def test_caps_far_above_the_scores(rows, dtype):
    """In float32 a score keeps its own precision under a cap of any size; an infinite one is none."""
    f = Filled([100, 150], 2, 64, 16, 8)
    q = query(2 if rows is None else sum(rows), 4, 64, dtype)
    for cap in (65.0, 1024.0) + ((1e4, 1e7, 2.0 ** 64) if dtype == torch.float32 else ()):
        f.check(q, rows, softcap=cap)
    assert torch.equal(f.attend(q, rows, softcap=float("inf")), f.attend(q, rows))


def test_more_rows_are_allowed_than_there_are():
    f = Filled([40] * 8, 1, 64, 16, 8)
    q = query(8, 8, 64, torch.bfloat16)
    want = f.attend(q)
    for most in (8, 1 << 29, 2 ** 31 - 1):
        assert torch.equal(f.attend(q, [1] * 8, max_rows=most), f.attend(q, [1] * 8, max_rows=8))
    f.check(q, [1] * 8, max_rows=1 << 29)
    assert torch.equal(f.attend(q, [1] * 8, max_rows=1), want)


@pytest.mark.parametrize("rows", [[5, 0, 9], [64, 3, 70]])
def test_more_rows_than_tokens_and_rows_behind_the_last_sequence(rows):
    """Rows that stand before the first token are zero; rows of no sequence stay as they were."""
    f = Filled([2, 7, 9], 1, 64, 16, 8)
    n = sum(rows)
    q = query(n + 6, 2, 64, torch.bfloat16)
    out = torch.full_like(q, 3.0)
    assert f.check(q, rows, out=out) is out
    assert (out[n:] == 3.0).all()
    assert not out[: rows[0] - 2].any()
    # of each sequence no more than max_rows
    # (a call of fewer rows may take another kernel: both are within the bound of the same 64-bit values)
    part = f.attend(q, rows, out=torch.full_like(q, 5.0), max_rows=4)
    want, bound = ref.attention(q, f.k, f.v, f.lengths, np.cumsum([0] + rows), 0.125, terms=1, dtype=torch.bfloat16)
    at = 0
    for r in rows:
        done = slice(at, at + min(r, 4))
        assert (np.abs(ref.f64(part[done]) - want[done]) <= bound[done]).all()
        assert (part[at + min(r, 4):at + r] == 5.0).all()
        at += r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("rows", [8, 70])
def test_nan_and_infinity_reach_the_rows_that_see_them_alone(rows, bits, dtype):
    n = 100
    f = Filled([n], 1, 64, 16, bits)
    q = query(rows, 2, 64, dtype)
    clean = f.attend(q, [rows])
    k, v = torch.randn(n, 1, 64), torch.randn(n, 1, 64)
    k, v = torch.from_numpy(f.k[0]).float(), torch.from_numpy(f.v[0]).float()
    k[n - 2, 0, 3] = float("inf")
    f.put(0, k, v)
    out = f.attend(q, [rows])
    assert torch.isnan(out[-2:]).all() and torch.equal(out[:-2], clean[:-2])
    k[n - 2, 0, 3] = 0.0
    v[n - 3, 0, 40] = float("nan")
    f.put(0, k, v)
    out = f.attend(q, [rows])
    assert torch.isnan(out[-3:, :, 32:]).all() and not torch.isnan(out[-3:, :, :32]).any()
    assert torch.equal(out[:-3], clean[:-3])
    # and a window that has passed them
    far = f.attend(q, [rows], window=1)
    assert not torch.isnan(far[-2:]).any()
    # a query that is not finite
    bad = q.clone()
    bad[1, 1, 5] = float("nan")
    f.put(0, torch.from_numpy(f.k[0]).float(), torch.from_numpy(f.v[0]).float())
    out = f.attend(bad, [rows])
    assert torch.isnan(out[1, 1]).all()
    out[1, 1] = clean[1, 1]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 40])
def test_what_is_not_finite_far_below_the_largest_score(rows, dtype):
    """A token whose weight vanishes beside another share's still makes the rows that see it NaN; a query that is
    infinite makes its row NaN, though every score of it be minus infinity."""
    f = Filled([3000], 1, 64, 16, 8)
    k, v = torch.randn(3000, 1, 64) * 0.1, torch.randn(3000, 1, 64)
    k[:, 0, 0] = torch.where(torch.arange(3000) < 1500, -400.0, -1.0)
    v[7, 0, 40] = float("inf")
    f.put(0, k, v)
    q = query(rows, 1, 64, dtype)
    q[:, 0, 0] = 30.0
    out = f.attend(q, [rows])
    assert torch.isnan(out[:, :, 32:]).all() and torch.isfinite(out[:, :, :32]).all()
    v[7, 0, 40] = 0.0
    f.put(0, k, v)
    q[1, 0, 0] = float("inf")
    out = f.attend(q, [rows])
    assert torch.isnan(out[1]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[2:]).all()


class Many:
    """So many heads, or so wide a table, that the tiles are the large ones; some heads are checked."""

    def __init__(self, H, group, D, bits, dtype, lengths, rows, width):
        g = torch.Generator(device="cuda").manual_seed(11)
        self.H, self.group, self.D, self.dtype, self.lengths, self.rows = H, group, D, dtype, lengths, rows
        pages = [-(-n // 32) for n in lengths]
        self.cache = ops.KvCache(sum(pages), 32, H, D, bits=bits)
        self.table = torch.zeros(len(lengths), width // 32, dtype=torch.int32)
        self.slots, at = [], 0
        for b, n in enumerate(pages):
            self.table[b, :n] = torch.arange(at, at + n).flip(0)
            j = torch.arange(lengths[b])
            self.slots.append((self.table[b][j // 32].long() * 32 + j % 32).cuda())
            at += n
        self.k, self.v = ([torch.randn(n, H, D, device="cuda", generator=g) for n in lengths] for _ in range(2))
        self.put()
        self.q = torch.randn(sum(rows), H * group, D, device="cuda", generator=g).to(dtype)
        self.starts = np.cumsum([0] + list(rows))

    def put(self):
        for b, s in enumerate(self.slots):
            ops.gpu_kv_cache_write(self.cache, self.k[b], self.v[b], s)

    def attend(self, **kw):
        i32 = torch.int32
        return ops.gpu_kv_cache_attention(self.q, self.cache, self.table.cuda(), torch.tensor(self.lengths, dtype=i32).cuda(),
                                          q_starts=torch.tensor(self.starts, dtype=i32).cuda(), max_rows=max(self.rows), **kw)

    def check(self, **kw):
        out = self.attend(**kw)
        held = [ops.gpu_kv_cache_read(self.cache, s) for s in self.slots]
        slopes = kw.pop("slopes", None)
        for h in (0, self.H // 2 - 1, self.H - 1):
            mine = slice(h * self.group, (h + 1) * self.group)
            want, bound = ref.attention(self.q[:, mine], [ref.f64(k[:, h:h + 1]) for k, _ in held], [ref.f64(v[:, h:h + 1]) for _, v in held],
                                        self.lengths, self.starts, self.D ** -0.5, terms=TERMS[self.dtype], dtype=self.dtype,
                                        slopes=None if slopes is None else ref.f64(slopes[mine]), **kw)
            err = np.abs(ref.f64(out[:, mine]) - want)
            assert not np.isnan(err).any() and (err <= bound).all(), "head %d off by %g of %g" % (h, err.max(), bound[err == err.max()][0])
        return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("H,group,D,lengths,rows,width", [
    (8, 2, 96, [300, 150, 40], [130, 70, 3], 16384), (8, 2, 128, [300, 150, 40], [130, 70, 33], 16384),  # shares, most of them empty
    (4, 3, 256, [290, 61], [100, 61], 32768), (180, 1, 96, [300], [270], 320), (180, 1, 128, [300], [270], 320),  # one share
    (180, 1, 224, [200, 140], [200, 140], 224), (200, 1, 64, [300, 30], [200, 30], 320),
    (256, 1, 64, [400, 100], [300, 20], 4096), (256, 1, 96, [400, 100], [300, 20], 4096), (180, 2, 128, [400], [300], 4096)])  # 8 waves
def test_large_tiles(H, group, D, lengths, rows, width, bits, dtype):
    m = Many(H, group, D, bits, dtype, lengths, rows, width)
    clean = m.check()
    m.check(window=70, softcap=20.0, slopes=torch.exp2(-torch.arange(1, H * group + 1).float() % 8).cuda())
    if bits == 4:
        m.check(causal=False)
    # a value that is not finite, in the first sequence's third token from the end
    m.v[0][-3, H - 1, 33] = float("nan")
    m.put()
    out, end = m.attend(), rows[0]
    last = slice((H - 1) * group, H * group)
    assert torch.isnan(out[end - 3:end, last, 32:64]).all()
    out[end - 3:end, last, 32:64] = clean[end - 3:end, last, 32:64]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("rows", [None, [3, 40]])
def test_pages_outside_the_cache_are_not_seen(rows):
    f = Filled([100, 90], 2, 64, 16, 4)
    f.table[0, 2] = -5
    f.table[1, 1] = 1 << 30
    n = 2 if rows is None else sum(rows)
    q = query(n, 4, 64, torch.float32)
    out = f.attend(q, rows)
    absent = [np.zeros(100, bool), np.zeros(90, bool)]
    absent[0][32:48] = True
    absent[1][16:32] = True
    starts = [0, 1, 2] if rows is None else [0, 3, 43]
    want, bound = ref.attention(q, f.k, f.v, f.lengths, starts, 0.125, absent=absent)
    assert (np.abs(ref.f64(out) - want) <= bound).all()


def test_lengths_and_starts_out_of_range_are_cut():
    """A length past the table's pages counts as far as they go, a negative one as none; starts that run
    backwards or past q name no row."""
    f = Filled([48, 48, 48], 1, 64, 16, 8)
    q = query(6, 2, 64, torch.bfloat16)
    table = f.table.cuda()

    def run(lengths, starts=None, q=q):
        return ops.gpu_kv_cache_attention(q, f.cache, table, torch.tensor(lengths, dtype=torch.int32).cuda(), out=torch.full_like(q, 2.0),
                                          q_starts=None if starts is None else torch.tensor(starts, dtype=torch.int32).cuda())

    a, b = run([48, 48, 48], q=q[:3]), run([1 << 30, 48, -7], q=q[:3])
    assert torch.equal(a[:2], b[:2]) and not b[2].any()
    out = run([48, 48, 48], [0, 2, 1, 99])
    want = run([48, 48, 48], [0, 2, 2, 2])
    assert torch.equal(out[:1], want[:1])
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("rows", [None, [20, 30]])
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_queries_and_outputs(rows, dtype):
    f = Filled([70, 60], 2, 96, 16, 4, spare=1)
    n = 2 if rows is None else sum(rows)
    wide = query(n, 3 * 4, 96, dtype)
    flat = torch.randn(n, 4 * 96 + 5, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    for q in (wide[:, 4:8], flat[:, 3:3 + 384].unflatten(1, (4, 96)), query(4, n, 96, dtype).transpose(0, 1)):
        want = f.attend(q.contiguous(), rows)
        out = torch.zeros(n, 9, 96, dtype=dtype, device="cuda")
        f.attend(q, rows, out=out[:, 2:6])
        assert torch.equal(out[:, 2:6], want) and not out[:, :2].any() and not out[:, 6:].any()
    # a table that is a slice of a wider one
    wide_table = torch.full((2, 40), -1, dtype=torch.int32)
    wide_table[:, : f.table.shape[1]] = f.table
    f.table = wide_table[:, : f.table.shape[1]]
    assert torch.equal(f.attend(q, rows), want)


@pytest.mark.parametrize("rows", [1, 60])
def test_captured_and_replayed_as_the_sequences_grow(rows):
    """One graph: a step is written and attended to, lengths and slots changing on the device between replays."""
    H, Hkv, D, page, B = 8, 2, 64, 16, 3
    width = 24
    cache = ops.KvCache(B * width, page, Hkv, D, bits=4)
    table = torch.arange(B * width, dtype=torch.int32).view(B, width).cuda()
    lengths = torch.zeros(B, dtype=torch.int32).cuda()
    slots = torch.zeros(B * rows, dtype=torch.int64).cuda()
    starts = (torch.arange(B + 1, dtype=torch.int32) * rows).cuda()
    k, v, q = (torch.zeros(B * rows, h, D, dtype=torch.bfloat16).cuda() for h in (Hkv, Hkv, H))

    def step(cache):
        ops.gpu_kv_cache_write(cache, k, v, slots)
        return ops.gpu_kv_cache_attention(q, cache, table, lengths, q_starts=starts if rows > 1 else None, max_rows=rows)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        slots.fill_(-1)
        step(cache)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(cache)
    other = ops.KvCache(B * width, page, Hkv, D, bits=4)
    at = torch.tensor([0, 17, 200])
    for n in range(3):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(n)))
        j = (at[:, None] + torch.arange(rows)).flatten()
        slots.copy_(torch.arange(B).repeat_interleave(rows) * width * page + j)
        at += rows
        lengths.copy_(at)
        graph.replay()
        torch.cuda.synchronize()
        want = step(other)
        torch.cuda.synchronize()
        assert torch.equal(cache.data, other.data) and torch.equal(got, want), n


def test_two_streams_at_once():
    f = Filled([900, 700], 2, 128, 16, 4)
    q = query(2, 8, 128, torch.bfloat16)
    want = f.attend(q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(f.attend(q))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_two_captured_calls_replayed_at_once():
    """Two graphs of calls with shares to join, replayed on two streams and beside eager calls: none meets another's
    workspace."""
    fs = [Filled([2500, 1700], 2, 128, 16, 4, seed=s) for s in (0, 1)]
    q = query(2, 8, 128, torch.bfloat16)
    want = [f.attend(q) for f in fs]
    side, graphs, outs = [torch.cuda.Stream() for _ in fs], [], []
    args = [(f.table.cuda(), torch.tensor(f.lengths, dtype=torch.int32).cuda()) for f in fs]
    torch.cuda.synchronize()
    for f, s, a in zip(fs, side, args):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(ops.gpu_kv_cache_attention(q, f.cache, *a))
        graphs.append(g)
    for n in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        eager = fs[0].attend(q)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and all(torch.equal(o, w) for o, w in zip(outs, want)), n


@pytest.mark.parametrize("rows", [None, [50]])
def test_a_cache_past_four_gigabytes(rows):
    pages, page, H, D = 1100, 1024, 8, 256
    cache = ops.KvCache(pages, page, H, D, bits=8)
    assert cache.data.numel() > 1 << 32
    n = 1500
    k, v = some((n, H, D), torch.bfloat16, 3, spread=0), some((n, H, D), torch.bfloat16, 4, spread=0)
    slots = torch.arange(pages * page - n, pages * page).cuda()
    ops.gpu_kv_cache_write(cache, k, v, slots)
    rk, rv = ops.gpu_kv_cache_read(cache, slots, dtype=torch.bfloat16)
    small = ops.KvCache(2, 1024, H, D, bits=8)
    at = torch.arange(2048 - n, 2048).cuda()
    ops.gpu_kv_cache_write(small, k, v, at)
    sk, sv = ops.gpu_kv_cache_read(small, at, dtype=torch.bfloat16)
    assert torch.equal(rk, sk) and torch.equal(rv, sv) and rk.any()
    q = query(1 if rows is None else rows[0], H, D, torch.bfloat16)

    def run(c, first):
        starts = None if rows is None else torch.tensor([0, rows[0]], dtype=torch.int32).cuda()
        return ops.gpu_kv_cache_attention(q, c, torch.tensor([[first, first + 1]], dtype=torch.int32).cuda(),
                                          torch.tensor([2048], dtype=torch.int32).cuda(), q_starts=starts, window=n - 50)

    assert torch.equal(run(cache, pages - 2), run(small, 0))


@pytest.mark.parametrize("bits", [4, 8])
def test_a_read_larger_than_the_gpus_caches(bits):
    H, D, n = 16, 128, 40000
    cache = ops.KvCache(n // 16 + 3, 16, H, D, bits=bits)
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(n, H, D, device="cuda", generator=g) for _ in range(2))
    slots = torch.arange(n, device="cuda") + 21
    slots[5000:5003] = -1
    ops.gpu_kv_cache_write(cache, k, v, slots)
    rk, rv = ops.gpu_kv_cache_read(cache, slots)
    for a in range(0, n, 1000):
        sk, sv = ops.gpu_kv_cache_read(cache, slots[a:a + 1000])
        assert torch.equal(rk[a:a + 1000], sk) and torch.equal(rv[a:a + 1000], sv)


def test_a_cache_keeps_its_memory():
    cache = ops.KvCache(4, 16, 2, 64)
    with pytest.raises(AttributeError):
        cache.data = cache.data.clone()
    other = ops.KvCache(4, 16, 2, 64)
    k = torch.randn(5, 2, 64).cuda()
    slots = torch.arange(5).cuda()
    ops.gpu_kv_cache_write(cache, k, k, slots)
    other.data.copy_(cache.data)
    assert torch.equal(ops.gpu_kv_cache_read(other, slots)[0], ops.gpu_kv_cache_read(cache, slots)[0])


@pytest.mark.parametrize("T", [40, 4100])
def test_slots_named_twice_harm_no_others(T):
    cache = ops.KvCache(T // 16 + 2, 16, 8, 32)
    k = torch.randn(T, 8, 32).cuda()
    slots = torch.arange(T).cuda()
    ops.gpu_kv_cache_write(cache, k, k, slots)
    want = ops.gpu_kv_cache_read(cache, slots)[0]
    twice = slots.clone()
    twice[T - 3:] = 7
    ops.gpu_kv_cache_write(cache, k, k, twice)
    got = ops.gpu_kv_cache_read(cache, slots)[0]
    keep = slots != 7
    assert torch.equal(got[keep], want[keep])


def test_refusals():
    cache = ops.KvCache(4, 16, 2, 64)
    k = torch.randn(3, 2, 64).cuda()
    slots = torch.arange(3).cuda()
    q = torch.randn(2, 4, 64).cuda()
    table = torch.zeros(2, 2, dtype=torch.int32).cuda()
    lengths = torch.ones(2, dtype=torch.int32).cuda()
    starts = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    att = ops.gpu_kv_cache_attention
    bad = [lambda: ops.KvCache(4, 16, 2, 64, bits=2), lambda: ops.KvCache(4, 20, 2, 64), lambda: ops.KvCache(4, 16, 2, 48),
           lambda: ops.KvCache(0, 16, 2, 64), lambda: ops.KvCache(4, 16, 2, 288), lambda: ops.KvCache(4, 2048, 2, 64),
           lambda: ops.gpu_kv_cache_write(cache, k, k[:2], slots), lambda: ops.gpu_kv_cache_write(cache, k, k.half(), slots),
           lambda: ops.gpu_kv_cache_write(cache, k.double(), k.double(), slots), lambda: ops.gpu_kv_cache_write(cache, k, k, slots.float()),
           lambda: ops.gpu_kv_cache_write(cache, k, k, slots[:2]), lambda: ops.gpu_kv_cache_write(cache, k[:, :1], k[:, :1], slots),
           lambda: ops.gpu_kv_cache_write(cache, k.cpu(), k, slots), lambda: ops.gpu_kv_cache_read(cache, slots, dtype=torch.float64),
           lambda: ops.gpu_kv_cache_read(cache, slots.view(1, 3)), lambda: ops.gpu_kv_cache_read(cache, slots.cpu()),
           lambda: att(q[:, :3], cache, table, lengths), lambda: att(q[:1], cache, table, lengths),
           lambda: att(q.double(), cache, table, lengths), lambda: att(q, cache, table.long(), lengths),
           lambda: att(q, cache, table[:1], lengths), lambda: att(q, cache, table, lengths, q_starts=starts[:2]),
           lambda: att(q, cache, table, lengths, softcap=-1.0), lambda: att(q, cache, table, lengths, window=-1),
           lambda: att(q, cache, table, lengths, slopes=torch.ones(3).cuda()), lambda: att(q[..., :32], cache, table, lengths),
           lambda: att(q, cache, table, lengths, out=q.half()), lambda: att(q, cache, table.cpu(), lengths),
           lambda: att(q, cache, table, lengths, softcap=float("nan")), lambda: att(q, cache, table, lengths, q_starts=starts, max_rows=-1)]
    for n, f in enumerate(bad):
        with pytest.raises(ops.IconnxError):
            f()
            pytest.fail("call %d was taken" % n)
