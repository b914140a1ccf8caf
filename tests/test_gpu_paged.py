"""Paged cache on the GPU: append (norm, rotation, K / V into pages), attention of drafted
trees and tree acceptance, against plain 64-bit forms.  Unused cache positions hold NaN and
unused table entries point nowhere, so a read of either shows."""
import numpy as np
import pytest

from rapidllm_amd import hip, ops
from rapidllm_amd.hip import DeviceBuffer, call
from rapidllm_amd.ops import BF16, F16, F32

pytestmark = pytest.mark.gpu

HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def rounded(a, dtype):
    return ops.row_values(ops.row_bits(a, dtype), dtype)


def cache_type(dtype):
    return BF16 if dtype == BF16 else F16


# ---------------------------------------------------------------- append


def norm_rope(x, gamma, pos, rot, theta, eps=1e-6, norm=True):
    """(result, scale of its error): x [rows][heads][hd] in 64 bits."""
    x = x.astype(np.float64)
    if norm:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if gamma is not None:
            x = x * (1.0 + gamma.astype(np.float64))
    half = rot // 2
    size = np.abs(x)
    if half:
        ang = np.asarray(pos, np.float64)[:, None] * float(theta) ** (-np.arange(half) / half)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        a, b = x[..., :half].copy(), x[..., half:rot].copy()
        x[..., :half], x[..., half:rot] = a * c - b * s, a * s + b * c
        size[..., :half] = size[..., half:rot] = np.abs(a) + np.abs(b)
    return x, size


def check(got, want, size, dtype):
    # 32-bit steps before the one rounding: the mean of squares of up to 256 values (a tree of 10
    # sums and the squares: 12 half steps, halved by the root), root, quotient, 3 products, cos or sin of
    # an angle known to pi half steps (5), products and sum of the turn (3): below 32 half steps
    tol = 32 * 2.0 ** -24 * size + HALF_STEP[dtype] * np.abs(want) * 1.01
    if dtype == F16:
        tol = tol + 2.0 ** -25  # half a step of the smallest values
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("dtype,nq,nkv,hd,rot,page,rows", [
    (F32, 24, 4, 256, 64, 16, 1), (F32, 24, 4, 256, 64, 256, 37), (F16, 5, 1, 128, 128, 1, 19),
    (BF16, 6, 2, 64, 16, 32, 130), (BF16, 32, 8, 128, 128, 64, 33), (F32, 1, 1, 64, 64, 8, 3),
    (F16, 8, 8, 256, 256, 128, 65), (F32, 3, 3, 128, 0, 4, 7), (F32, 40, 10, 128, 8, 16, 2500)])
@pytest.mark.parametrize("norm", [True, False])
def test_append(gpu, dtype, nq, nkv, hd, rot, page, rows, norm):
    r = np.random.default_rng(rows + hd + nq)
    n_pages = -(-rows // page) + 3
    cache = ops.PagedCache(n_pages, page, nkv, hd, cache_type(dtype), n_layers=2)
    before = [rounded(r.standard_normal(cache.shape), cache.desc.dtype) for _ in range(2)]
    cache.fill(*before)
    q, k, v = (rounded(r.standard_normal((rows, h, hd)) * 1.5, dtype) for h in (nq, nkv, nkv))
    qn, kn = (r.standard_normal(hd).astype(np.float32) * 0.2 for _ in range(2))
    pos = r.integers(0, 200000, rows)
    slots = r.permutation(n_pages * page)[:rows].astype(np.int64)
    left_out = r.random(rows) < 0.1  # rows without a slot, below and above the cache
    slots[left_out] = np.where(r.random(left_out.sum()) < 0.5, -1, n_pages * page + r.integers(0, 1 << 40))
    got = ops.paged_append(cache, 1, q, k, v, pos, slots, qn, kn, norm, 1e-6, rot, 5e5, dtype)
    check(got, *norm_rope(q, qn, pos, rot, 5e5, norm=norm), dtype)
    K, V = cache.values()
    want_k, size_k = norm_rope(k, kn, pos, rot, 5e5, norm=norm)
    at = slots[~left_out]
    check(K[1, at // page, :, at % page], want_k[~left_out], size_k[~left_out], cache.desc.dtype)
    assert np.array_equal(V[1, at // page, :, at % page], rounded(v[~left_out], cache.desc.dtype))
    # every other position is as it was
    keep = np.ones((2, n_pages, page), bool)
    keep[1, at // page, at % page] = False
    for now, old in ((K, before[0]), (V, before[1])):
        assert np.array_equal(now.transpose(0, 1, 3, 2, 4)[keep], old.transpose(0, 1, 3, 2, 4)[keep])


def test_append_rows_of_a_fused_projection(gpu):
    """q | gate interleaved per head, then k, v in one row (the strides the model's projection
    has), no norm weights, and keys alone (n_q = 0)."""
    r = np.random.default_rng(5)
    n, nq, nkv, hd = 9, 10, 2, 256
    Y = r.standard_normal((n, (2 * nq + 2 * nkv) * hd + 4)).astype(np.float32)  # rows 4 floats apart
    pos, slots = np.arange(1000, 1000 + n), np.arange(n)
    heads = Y[:, :-4].reshape(n, 2 * nq + 2 * nkv, hd)
    d = DeviceBuffer.from_numpy(Y)
    d_pos, d_slots = DeviceBuffer.from_numpy(pos.astype(np.int32)), DeviceBuffer.from_numpy(slots.astype(np.int64))
    out = DeviceBuffer(4 * n * nq * hd)
    for with_q in (True, False):
        cache = ops.PagedCache(1, 16, nkv, hd)
        call("rl_hip_paged_append", cache.desc, 0, F32, d.ptr if with_q else None, Y.shape[1], 2 * hd,
             d.ptr + 4 * 2 * nq * hd, Y.shape[1], hd, d.ptr + 4 * (2 * nq + nkv) * hd, Y.shape[1], hd, None, None, 1,
             1e-6, 64, 1e7, d_pos.ptr, d_slots.ptr, n, nq if with_q else 0, out.ptr if with_q else None, None)
        K, V = cache.values()
        want, size = norm_rope(heads[:, 2 * nq:2 * nq + nkv], None, pos, 64, 1e7)
        check(K[0, 0, :, :n].transpose(1, 0, 2), want, size, F16)
        assert np.array_equal(V[0, 0, :, :n].transpose(1, 0, 2), rounded(heads[:, 2 * nq + nkv:], F16))
    check(out.numpy(np.float32, (n, nq, hd)), *norm_rope(heads[:, :2 * nq:2], None, pos, 64, 1e7), F32)


def test_append_far_positions(gpu):
    """Angles at positions that 32-bit arithmetic cannot turn by."""
    r = np.random.default_rng(8)
    pos = np.array([0, 1, 1 << 20, (1 << 24) + 1, (1 << 31) - 1])
    q = r.standard_normal((5, 2, 128)).astype(np.float32)
    cache = ops.PagedCache(1, 8, 1, 128)
    got = ops.paged_append(cache, 0, q, q[:, :1], q[:, :1], pos, np.arange(5), rotary_dim=128, theta=1e4)
    # 64-bit angles up to 2^31: theta^(-2i/rot) and its product are off by a few 2^-53 of 2^31 radians
    want, size = norm_rope(q, None, pos, 128, 1e4)
    check(got, want, size * (1 + 2.0 ** -18 / 2.0 ** -24 / 32), F32)


# ---------------------------------------------------------------- attention


class Step:
    """Sequences in random pages, NaN wherever no sequence has a position."""

    def __init__(self, seed, dtype, nq, nkv, hd, page, ctx, rows, spare=2, kstd=1.0):
        r = self.r = np.random.default_rng(seed)
        self.dtype, self.nq, self.nkv, self.hd, self.page, self.ctx, self.rows = dtype, nq, nkv, hd, page, ctx, rows
        ct = cache_type(dtype)
        need = [-(-(c + n) // page) for c, n in zip(ctx, rows)]
        order = r.permutation(sum(need) + spare)
        self.table = np.where(r.random((len(ctx), max(need) + 2)) < 0.5, -1, 1 << 30).astype(np.int32)
        self.cache = ops.PagedCache(sum(need) + spare, page, nkv, hd, ct)
        self.K, self.V = (np.full(self.cache.shape, np.nan, np.float32) for _ in range(2))
        self.kv, at = [], 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
            L = ctx[b] + rows[b]
            kv = [rounded(r.standard_normal((L, nkv, hd)) * kstd, ct) for _ in range(2)]
            self.kv.append(kv)
            p = np.arange(L)
            for pool, x in ((self.K, kv[0]), (self.V, kv[1])):
                pool[0, self.table[b][p // page], :, p % page] = x
        self.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        n = int(self.start[-1])
        self.q = rounded(r.standard_normal((n, nq, hd)) * 1.5, dtype)
        self.gate = rounded(r.standard_normal((n, nq, hd)), dtype)
        self.cache.fill(self.K, self.V)

    def tree_mask(self, words=None, drop=0.0):
        """Ancestors' bits of random trees; some rows see nothing of the tree, not even themselves."""
        R = max(self.rows + [1])
        words = words or -(-R // 64)
        mask = np.zeros((int(self.start[-1]), words), np.uint64)
        for b, n in enumerate(self.rows):
            bits = []
            for i in range(n):
                up = bits[int(self.r.integers(max(0, i - 5), i))] if i else 0
                bits.append(up | 1 << i)
            for i in range(n):
                v = 0 if self.r.random() < drop else bits[i]
                for w in range(words):
                    mask[self.start[b] + i, w] = (v >> (64 * w)) & ((1 << 64) - 1)
        return mask

    def want(self, mask, gate, scale=None):
        """(result, tolerance) per row in 64 bits."""
        scale = 1 / np.sqrt(self.hd) if scale is None else scale
        G = self.nq // self.nkv
        out, tol = np.zeros(self.q.shape), np.zeros(self.q.shape)
        for b, (c, n) in enumerate(zip(self.ctx, self.rows)):
            k, v = (x.astype(np.float64) for x in self.kv[b])
            for j in range(n):
                row = self.start[b] + j
                sees = np.ones(c + n, bool)
                for i in range(n):
                    sees[c + i] = i <= j if mask is None else \
                        i // 64 < mask.shape[1] and bool(int(mask[row, i // 64]) >> (i % 64) & 1)
                if not sees.any():
                    continue
                for h in range(self.nq):
                    kk, vv, q = k[sees, h // G], v[sees, h // G], self.q[row, h].astype(np.float64)
                    s = kk @ q * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    o, A = p @ vv, p @ np.abs(vv)
                    # a score is off by its dot product's 32-bit sum (32 steps) and, from 32-bit rows, by the
                    # 2^-22 that two half-precision parts leave; a weight by twice that, its own rounding and the
                    # exponential's; the sums over positions by a step in 16 positions
                    part = 2.0 ** -22 if self.dtype == F32 else 0.0
                    S = np.abs(scale) * (np.abs(kk) @ np.abs(q)).max()
                    rel = 2 * S * (32 * 2.0 ** -24 + part) + (64 + sees.sum() / 16) * 2.0 ** -24 + \
                        (part or HALF_STEP[self.dtype])
                    t = A * rel
                    if gate:
                        g = 1 / (1 + np.exp(-self.gate[row, h].astype(np.float64)))
                        o, t = o * g, t * g + 4 * 2.0 ** -24 * np.abs(o * g)
                    out[row, h] = o
                    tol[row, h] = t + 1.01 * HALF_STEP[self.dtype] * np.abs(o) + (2.0 ** -25 if self.dtype == F16 else 0)
        return out, tol

    def run(self, mask=None, gate=False, scale=None, **kw):
        return ops.tree_attn(self.cache, 0, self.q, self.table, self.ctx, self.start, mask,
                             self.gate if gate else None, scale, self.dtype, **kw)


def agree(got, want, tol):
    assert np.all(np.isfinite(got))
    bad = np.abs(got - want) / np.maximum(tol, 1e-30)
    assert np.all(bad <= 1), (bad.max(), np.unravel_index(bad.argmax(), bad.shape))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("nq,nkv,hd,page,ctx,rows", [
    (24, 4, 256, 16, [0], [1]), (24, 4, 256, 16, [700], [1]), (10, 2, 256, 64, [63, 64, 65], [1, 2, 3]),
    (5, 1, 256, 1, [31, 0, 200], [9, 4, 1]), (32, 8, 128, 32, [1000, 3, 129, 513], [8, 1, 0, 5]),
    (16, 16, 128, 128, [127, 300], [3, 17]), (8, 8, 64, 256, [255, 256, 257], [1, 1, 1]),
    (6, 2, 64, 2, [61], [70]), (64, 1, 128, 16, [90], [3]), (24, 4, 256, 256, [1500], [64]),
    (4, 4, 128, 4096, [70, 10], [33, 2])])
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_tree_attn(gpu, dtype, nq, nkv, hd, page, ctx, rows, kind):
    s = Step(len(ctx) * 100 + hd + nq + page, dtype, nq, nkv, hd, page, ctx, rows)
    mask = s.tree_mask() if kind == "tree" else None
    gate = kind == "tree"
    got = s.run(mask, gate)
    agree(got, *s.want(mask, gate))
    assert np.array_equal(got, s.run(mask, gate))  # the same from call to call


@pytest.mark.parametrize("hd,nq,nkv,rows", [(64, 4, 2, 3), (64, 12, 1, 5), (128, 8, 2, 9), (128, 8, 1, 20),
                                            (256, 4, 1, 2), (256, 6, 1, 10), (256, 6, 1, 30)])
@pytest.mark.parametrize("page", [1, 2, 4, 8, 32])
def test_small_pages_under_long_contexts(gpu, hd, nq, nkv, rows, page):
    """Every way a tile's rows are found, over many tiles: each row by itself, runs of rows, whole tiles."""
    s = Step(page + hd, F16 if page % 4 else F32, nq, nkv, hd, page, [1900, 130, 1500], [rows, 1, rows])
    mask = s.tree_mask()
    agree(s.run(mask), *s.want(mask, False))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_see_nothing(gpu, dtype):
    """A mask without a bit: zeros where the context is empty too, the context alone where not."""
    s = Step(3, dtype, 8, 2, 128, 16, [0, 40, 0], [6, 7, 33])
    mask = s.tree_mask(drop=0.5)
    mask[0] = 0
    got = s.run(mask)
    agree(got, *s.want(mask, False))
    assert not got[0].any()
    for row in list(range(6)) + list(range(13, 46)):
        assert mask[row].any() or not got[row].any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("R", [7, 40])
def test_what_a_row_does_not_see_does_not_reach_it(gpu, dtype, R):
    """K and V of some drafted tokens are infinite or NaN: rows that see none of them are as exact
    as before, rows that see one get what the sum has."""
    s = Step(R, dtype, 12, 4, 128, 16, [0, 75, 130], [R, R, 1])
    mask = s.tree_mask()
    want, tol = s.want(mask, False)
    poison = {2: np.nan, 3: np.inf, 5: -np.inf}
    for b in (0, 1):
        for j, x in poison.items():
            p = s.ctx[b] + j
            s.K[0, s.table[b, p // 16], :, p % 16, ::3] = x
            s.V[0, s.table[b, p // 16], :, p % 16, ::5] = x
    s.cache.fill(s.K, s.V)
    got = s.run(mask)
    hit = np.array([any(int(mask[i, 0]) >> j & 1 for j in poison) for i in range(len(mask))])
    hit[s.start[2]:] = False
    assert 0 < hit.sum() < len(hit)
    agree(got[~hit], want[~hit], tol[~hit])
    sees_nan = np.array([bool(int(mask[i, 0]) >> 2 & 1) for i in range(len(mask))]) & hit
    assert np.isnan(got[sees_nan]).all()


def test_infinite_v_where_it_is_seen(gpu):
    """Finite keys, an infinity in one dim of a drafted token's V: that dim becomes infinite for the
    rows that see it, and nothing else changes."""
    s = Step(11, F32, 4, 2, 64, 16, [50], [10])
    mask = s.tree_mask()
    want, tol = s.want(mask, False)
    p = s.ctx[0] + 4
    s.V[0, s.table[0, p // 16], :, p % 16, 7] = np.inf
    s.cache.fill(s.K, s.V)
    got = s.run(mask)
    sees = np.array([bool(int(m) >> 4 & 1) for m in mask[:, 0]])
    assert np.isposinf(got[sees][..., 7]).all()
    got[sees, :, 7] = want[sees, :, 7]
    agree(got, want, tol)


def test_large_scores(gpu):
    """Scores of thousands: the running maximum takes them."""
    s = Step(21, F32, 4, 2, 128, 16, [300], [5], kstd=1.0)
    for scale in (40.0, -40.0, 0.0):
        got = s.run(None, scale=scale)
        agree(got, *s.want(None, False, scale))


def test_rows_behind_the_last_sequence_and_past_max_rows(gpu):
    s = Step(31, BF16, 8, 2, 64, 32, [100, 20], [3, 2])
    n = 5
    s.q = rounded(s.r.standard_normal((n + 4, 8, 64)), BF16)
    old = rounded(s.r.standard_normal((n + 4, 8, 64)), BF16)
    got = s.run(out0=old)
    assert np.array_equal(got[n:], old[n:])
    full = got.copy()
    s.q = s.q[:n + 4]
    got = s.run(out0=old, max_rows=2)  # sequence 0 has three rows
    assert np.array_equal(got[2], old[2])
    s.q = s.q[:n]
    want, tol = s.want(None, False)
    agree(full[:n], want, tol)


def test_lengths_and_pages_that_make_no_sense(gpu):
    """Negative or too long contexts are cut to the table, pages outside the cache are page 0, and the
    other sequence is not touched by either."""
    s = Step(41, F32, 4, 2, 128, 16, [33, 50], [2, 3], spare=3)
    s.K = np.nan_to_num(s.K)
    s.V = np.nan_to_num(s.V)
    s.cache.fill(s.K, s.V)
    want, tol = s.want(None, False)
    table = s.table
    for ctx0, bad in ((-5, 0), (1 << 30, -7), (33, 1 << 30), (33, -(1 << 31))):
        t = table.copy()
        t[0, 1] = bad
        t[0, 4:] = bad
        got = ops.tree_attn(s.cache, 0, s.q, t, [ctx0, 50], s.start)
        agree(got[2:], want[2:], tol[2:])
    # row_start that goes back or past the rows
    got = ops.tree_attn(s.cache, 0, s.q, table, [33, 50], [0, 5, 900], max_rows=5)
    assert got.shape == s.q.shape


def test_strided_rows_and_gates(gpu):
    """q and gate interleaved in the projection's rows, as the model has them."""
    s = Step(51, F32, 6, 2, 256, 16, [70], [4])
    n, nq, hd = s.q.shape
    Y = np.zeros((n, nq * 2 * hd + 8), np.float32)
    Y[:, :-8].reshape(n, nq, 2, hd)[:, :, 0] = s.q
    Y[:, :-8].reshape(n, nq, 2, hd)[:, :, 1] = s.gate
    d, t, c, st = (DeviceBuffer.from_numpy(a) for a in (Y, s.table, np.int32(s.ctx), s.start))
    out = DeviceBuffer(4 * n * nq * hd)
    ws = DeviceBuffer(hip.lib().rl_hip_tree_attn_workspace_bytes(nq, 2, hd, 1, 4))
    call("rl_hip_tree_attn", s.cache.desc, 0, F32, d.ptr, Y.shape[1], 2 * hd, d.ptr + 4 * hd, Y.shape[1], 2 * hd, t.ptr,
         s.table.shape[1], c.ptr, st.ptr, 1, n, 4, None, 0, nq, hd ** -0.5, out.ptr, ws.ptr, ws.nbytes, None)
    agree(out.numpy(np.float32, (n, nq, hd)), *s.want(None, True))


def test_cache_past_32_bit_offsets(gpu):
    """Pages whose elements lie past 2^32: appended to, attended and moved."""
    r = np.random.default_rng(61)
    nkv, hd, page, pages = 4, 256, 256, 16640  # 2^32 elements end at page 16384
    cache = ops.PagedCache(pages, page, nkv, hd)
    table = np.array([[pages - 1, 16383, pages - 2]], np.int32)
    n, ctx = 600, 0
    k, v = (rounded(r.standard_normal((n, nkv, hd)), F16) for _ in range(2))
    p = np.arange(n)
    slots = table[0][p // page].astype(np.int64) * page + p % page
    ops.paged_append(cache, 0, np.zeros((n, 4, hd)), k, v, p, slots, norm=False, rotary_dim=0)
    s = Step(62, F32, 8, nkv, hd, page, [n - 4], [4])
    s.cache, s.table, s.kv = cache, table, [[k, v]]
    agree(s.run(), *s.want(None, False))
    # path rows 0, 2, 3: position ctx + 1 takes row 2's, ctx + 2 row 3's
    path, acc, nxt, ctx_out = ops.tree_accept(cache, table, [n - 4], [0, 4], [-1, 0, 0, 2], [5, 6, 7, 8], [7, 9, 8, 3], 4)
    assert path.tolist() == [[0, 2, 3, -1]] and acc[0] == 3 and nxt[0] == 3 and ctx_out[0] == n - 1
    order = np.r_[0:n - 3, n - 2, n - 1, n - 1]
    s.kv = [[k[order], v[order]]]
    agree(s.run(), *s.want(None, False))


# ---------------------------------------------------------------- acceptance


def walk(parents, toks, samples, cap):
    path = [0] if len(parents) else []
    while path and len(path) < cap:
        fit = [j for j in range(len(parents)) if j > path[-1] and parents[j] == path[-1] and toks[j] == samples[path[-1]]]
        if not fit:
            break
        path.append(fit[0])
    return path


@pytest.mark.parametrize("dtype,hd,page,layers", [(F16, 256, 16, 1), (BF16, 128, 1, 3), (F16, 64, 128, 16)])
@pytest.mark.parametrize("rows,cap", [([1], 4), ([4, 9, 0, 64], 64), ([150, 3, 20], 9), ([300], 300)])
def test_tree_accept(gpu, dtype, hd, page, layers, rows, cap):
    r = np.random.default_rng(sum(rows) + hd)
    B, nkv, total = len(rows), 2, sum(rows)
    ctx = [int(r.integers(0, 70)) for _ in rows]
    need = [-(-(c + n) // page) for c, n in zip(ctx, rows)]
    order, at = r.permutation(sum(need) + 2), 0
    table = np.full((B, max(need) + 1), -1, np.int32)
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cache = ops.PagedCache(sum(need) + 2, page, nkv, hd, dtype, layers)
    K, V = (rounded(r.standard_normal(cache.shape), dtype) for _ in range(2))
    cache.fill(K, V)
    start = np.concatenate([[0], np.cumsum(rows)])
    parents = np.concatenate([[-1 if i == 0 else r.integers(max(0, i - 4), i) for i in range(n)] for n in rows]).astype(int)
    toks = r.integers(0, 6, total)
    samples = r.integers(0, 6, total)
    for b, n in enumerate(rows):  # most samples are some child's token
        for i in range(1, n):
            if r.random() < 0.8:
                samples[start[b] + parents[start[b] + i]] = toks[start[b] + i]
    path, acc, nxt, ctx_out = ops.tree_accept(cache, table, ctx, start, parents, toks, samples, cap)
    for b, n in enumerate(rows):
        sl = slice(start[b], start[b + 1])
        want = walk(parents[sl], toks[sl], samples[sl], cap)
        assert path[b].tolist() == want + [-1] * (cap - len(want))
        assert acc[b] == len(want) and ctx_out[b] == ctx[b] + len(want)
        assert nxt[b] == (samples[start[b] + want[-1]] if want else -1)
        old = [K.copy(), V.copy()]
        for d, j in enumerate(want):
            f, t = ctx[b] + j, ctx[b] + d
            for new, src in ((K, old[0]), (V, old[1])):
                new[:, table[b, t // page], :, t % page] = src[:, table[b, f // page], :, f % page]
    for got, want in zip(cache.values(), (K, V)):
        assert np.array_equal(got, want)


def test_accept_without_a_cache_and_with_bad_trees(gpu):
    """Parents at or past their own row have no children; no cache: the path alone."""
    parents = [3, 0, 1, 3, 2, 99]
    toks = [0, 1, 1, 1, 1, 1]
    samples = [1, 1, 1, 1, 4, 1]
    path, acc, nxt, ctx = ops.tree_accept(None, None, [10], [0, 6], parents, toks, samples, 8)
    assert path[0].tolist() == [0, 1, 2, 4, -1, -1, -1, -1] and acc[0] == 4 and nxt[0] == 4 and ctx[0] == 14


def test_accept_pages_outside_the_cache(gpu):
    """Rows on such pages are not moved; everything else is."""
    cache = ops.PagedCache(4, 2, 1, 64)
    K = np.arange(np.prod(cache.shape)).reshape(cache.shape) % 1024
    cache.fill(K, K + 1)
    # path rows 0, 2, 4 at positions 1, 3, 5: pages 0, 1, 2 of the table
    path, acc, _, _ = ops.tree_accept(cache, [[3, 1, 1 << 20]], [1], [0, 5], [-1, 0, 0, 0, 2], [1, 1, 2, 3, 5],
                                      [2, 0, 5, 0, 9], 5)
    assert path[0].tolist() == [0, 2, 4, -1, -1]
    want = K.copy()
    want[0, 1, :, 0] = K[0, 1, :, 1]  # position 2 takes row 2's (position 3); position 3 keeps its own
    for got, w in zip(cache.values(), (want, want + 1)):
        assert np.array_equal(got, w.astype(np.float32))
