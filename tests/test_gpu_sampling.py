"""Sampling on the GPU against a plain 64-bit form: the same token for the same random number, its
probability to 2^-20."""
import numpy as np
import pytest

from rapidllm_amd import ops
from rapidllm_amd.ops import BF16, F16, F32

pytestmark = pytest.mark.gpu


def plain(z, u, t=1.0, k=0, p=1.0, mp=0.0):
    """(token, probability, distance of u from the nearest border of its token's share)."""
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    top = int(np.argmax(z))
    if z[top] == -np.inf:
        return 0, 0.0, 1.0
    if not t > 0:
        return top, 1.0, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(z == z[top], 1.0, np.exp((z - z[top]) / float(t)))
    w[np.isnan(w) | (z == -np.inf)] = 0.0
    order = np.lexsort((np.arange(z.size), -z))
    if 0 < k < z.size:
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        order = order[:max(1, int((np.concatenate([[0.0], c[:-1]]) < float(p) * c[-1]).sum()))]
    keep = np.sort(order)
    if mp > 0:
        keep = keep[w[keep] >= min(float(mp), 1.0)]
    c = np.cumsum(w[keep])
    x = float(np.clip(u, 0, np.float32(1) - np.float32(2.0 ** -24))) * c[-1]
    j = int(np.searchsorted(c, x, side="right"))
    low = c[j] - w[keep[j]]
    return int(keep[j]), w[keep[j]] / c[-1], min(x - low, c[j] - x) / c[-1]


def check(z, u, dtype=F32, **kw):
    z = ops.row_values(ops.row_bits(z, dtype), dtype)
    z = np.atleast_2d(z)
    n = len(z)
    u = np.broadcast_to(np.float32(u), (n,))
    col = {a: np.broadcast_to(np.asarray(v, np.int32 if a == "top_k" else np.float32), (n,)) for a, v in kw.items()
           if a != "ld"}
    idx, prob = ops.sample_rows(z, u, dtype=dtype, **kw)
    for i in range(n):
        g = {a: v[i] for a, v in col.items()}
        want, pr, room = plain(z[i], u[i], g.get("temperature", 1.0), int(g.get("top_k", 0)), g.get("top_p", 1.0),
                               g.get("min_p", 0.0))
        # borders are known to 2^-45 of the largest weight a token: below 2^-27 of the total
        if want != idx[i] and 0 < room < 2.0 ** -26:
            continue
        assert idx[i] == want, (i, idx[i], want, room, g)
        # the probability: its own rounding, and half a unit (2^-45) in a weight of at least that
        assert abs(prob[i] - pr) <= 2.0 ** -20 * pr + 2.0 ** -40, (i, prob[i], pr, g)


def rows(seed, n, V, std=2.0):
    r = np.random.default_rng(seed)
    z = r.standard_normal((n, V)) * std
    z[np.arange(n)[:, None], r.integers(0, V, (n, 30))] += r.uniform(2, 12, (n, 30))
    return z.astype(np.float32), r.random(n).astype(np.float32), r


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("V,n", [(1, 3), (2, 9), (7, 20), (64, 30), (1000, 40), (1023, 9), (1025, 9), (32000, 20),
                                 (50257, 7), (248320, 24)])
def test_mixed_settings(gpu, dtype, V, n):
    z, u, r = rows(V + n, n, V)
    pick = lambda *v: r.choice(v, n)  # noqa: E731
    check(z, u, dtype, temperature=pick(0.0, 0.3, 0.7, 1.0, 1.3, 5.0), top_k=pick(0, 1, 2, 20, 50, 1000, V, V + 1),
          top_p=pick(1.0, 0.9, 0.95, 0.5, 0.05, 0.0, -1.0, 2.0), min_p=pick(0.0, 0.0, 0.02, 0.3, 1.0, 2.0, -1.0))


@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.8), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05),
                                dict(temperature=1.5, top_p=0.97), dict(top_k=5000, top_p=0.99),
                                dict(top_k=50, top_p=0.9, min_p=0.05, temperature=0.7)])
def test_each_setting_alone(gpu, kw):
    z, u, _ = rows(7, 12, 151936)
    check(z, u, **kw)


def test_one_row_of_many_numbers(gpu):
    """The whole distribution of a row: u on a grid, every token by its share."""
    z, _, _ = rows(9, 1, 3001)
    n = 512
    check(np.repeat(z, n, 0), (np.arange(n) / n).astype(np.float32), top_k=100, top_p=0.95)
    check(np.repeat(z, n, 0), (np.arange(n) / n).astype(np.float32), temperature=2.0)


def test_equal_logits(gpu):
    """Ties go to the lowest index: all equal, two values, and halves of 16-bit logits."""
    V = 30011
    flat = np.zeros((6, V), np.float32)
    u = np.array([0.0, 0.25, 0.5, 0.75, 0.99999994, 0.1], np.float32)
    check(flat, u)
    check(flat, u, top_k=[1, 2, 7, 1000, 30010, 5000])
    check(flat, u, top_p=[0.5, 0.25, 0.9, 0.0, 0.999, 0.125])
    check(flat, u, top_k=[9, 20000, 30000, 4097, 4096, 2], top_p=[0.5, 0.25, 0.9, 0.75, 0.999, 0.125])
    two = flat.copy()
    two[:, 1::3] = 1.0
    check(two, u, top_k=[5, 10003, 10004, 10005, 20000, 30000])
    check(two, u, top_p=[0.5, 0.3, 0.9, 0.6, 0.7, 0.58])
    r = np.random.default_rng(3)
    check(np.round(r.standard_normal((6, V)) * 4) / 4, u, BF16, top_p=[0.9, 0.5, 0.99, 0.8, 0.7, 0.6])
    signed = np.where(np.arange(V) % 2, -0.0, 0.0).astype(np.float32)
    check(np.tile(signed, (6, 1)), u, top_k=[1, 2, 3, 4, 5, 6])


def test_flat_logits_with_many_in_a_bin(gpu):
    """More elements around the border than shared memory puts in order, all different."""
    r = np.random.default_rng(4)
    z = (r.random((4, 248320)) * 1e-3).astype(np.float32)
    check(z, r.random(4), top_p=[0.9, 0.5, 0.999, 0.01])
    check(z, r.random(4), top_k=[5000, 100000, 1, 248319])
    check(z, r.random(4), top_k=[5000, 100000, 200000, 240000], top_p=0.7, temperature=[1.0, 1e6, 1e-5, 3.0])


def test_infinities_nans_and_masked_rows(gpu):
    r = np.random.default_rng(5)
    z = r.standard_normal((10, 5000)).astype(np.float32)
    z[0] = -np.inf
    z[1] = np.nan
    z[2, 100:] = -np.inf
    z[3, ::2] = np.nan
    z[4, [7, 4000, 4999]] = np.inf
    z[5] = -np.inf
    z[5, 4321] = -1e30
    z[6, 5] = np.inf
    z[6, 6] = np.nan
    z[7] = np.finfo(np.float32).min
    z[8] = np.finfo(np.float32).min
    z[8, 77] = np.finfo(np.float32).max
    u = r.random(10).astype(np.float32)
    check(z, u)
    check(z, u, temperature=0.0)
    check(z, u, top_k=3, top_p=0.6)
    check(z, u, top_p=0.9, min_p=0.2, temperature=0.5)


def test_numbers_and_settings_at_their_limits(gpu):
    z, _, _ = rows(11, 8, 4000)
    u = np.array([0.0, 1.0, -1.0, 2.0, np.nan, 0.99999994, 2.0 ** -24, 0.5], np.float32)
    uu = np.where(np.isnan(u), 0, u)
    for kw in (dict(), dict(top_k=7), dict(top_p=0.8), dict(temperature=1e-30), dict(temperature=1e30),
               dict(temperature=np.inf), dict(min_p=1.0)):
        got = ops.sample_rows(z, u, **kw)
        for i in range(8):
            want, pr, _ = plain(z[i], uu[i], kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0),
                                kw.get("min_p", 0.0))
            assert got[0][i] == want and abs(got[1][i] - pr) <= 2.0 ** -20 * pr + 2.0 ** -40, (kw, i)
    nan = np.float32(np.nan)
    a = ops.sample_rows(z, uu, top_p=nan, min_p=nan, top_k=-3)
    b = ops.sample_rows(z, uu)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    assert np.array_equal(ops.sample_rows(z, uu, temperature=nan)[0], z.argmax(1))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_rows_with_a_stride(gpu, dtype):
    z, u, _ = rows(13, 5, 999)
    check(z, u, dtype, ld=1007, top_k=20, top_p=0.9)


def test_the_same_from_call_to_call(gpu):
    z, u, _ = rows(15, 6, 100000, std=3.0)
    a = [ops.sample_rows(z, u, temperature=1.2, top_p=0.95) for _ in range(3)]
    for b in a[1:]:
        assert np.array_equal(a[0][0], b[0]) and np.array_equal(a[0][1], b[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_low_temperatures_and_far_apart_logits(gpu, dtype):
    """Top-k reaches logits that weigh nothing, deep below the maximum; rows of which little is left
    by a mask; more of top-k than logits above -infinity."""
    z, u, r = rows(17, 8, 40000, std=3.0)
    z[1, 300:] = -np.inf
    z[2, 20:] = -np.inf
    z[3] *= 1e4
    z[4, 7:] = -np.inf
    z[5] = np.where(r.random(40000) < 1e-3, z[5], -np.inf)
    for t in (0.01, 1e-6, 1e-30, 1.0, 1e4, np.inf):
        check(z, u, dtype, temperature=t, top_k=[50, 50, 50, 30, 10, 39, 700, 3000])
        check(z, u, dtype, temperature=t, top_k=[50, 500, 20, 3000, 10, 39, 0, 1], top_p=0.9, min_p=0.01)
        check(z, u, dtype, temperature=t, top_p=[0.5, 0.9, 0.99, 0.999, 0.1, 0.7, 0.3, 0.95])


def test_most_likely_tokens_side_by_side(gpu):
    """The largest logits in one run of indices: more of them in a tile than the tiles' maxima show."""
    r = np.random.default_rng(19)
    z = r.standard_normal((6, 248320)).astype(np.float32)
    z[:, 70000:76000] += 20
    u = r.random(6).astype(np.float32)
    check(z, u, top_k=[1, 40, 200, 240, 1500, 5500])
    check(z, u, top_k=[1, 40, 200, 240, 1500, 5500], top_p=0.9)
    check(z, u, top_p=[0.9, 0.99, 0.5, 0.1, 0.999, 0.97])


@pytest.mark.parametrize("V", [(1 << 20) + 3, 3000001])
def test_large_vocabularies(gpu, V):
    """Groups of several tiles, shares of several tiles per thread; coarser units."""
    r = np.random.default_rng(V)
    z = (r.standard_normal((3, V)) * 2).astype(np.float32)
    z[:, r.integers(0, V, 50)] += 9
    u = r.random(3).astype(np.float32)
    for kw in (dict(), dict(top_k=[40, 300, 3000]), dict(top_p=[0.9, 0.5, 0.99]), dict(temperature=0.0)):
        idx, prob = ops.sample_rows(z, u, **kw)
        for i in range(3):
            g = {a: np.broadcast_to(v, (3,))[i] for a, v in kw.items()}
            want, pr, room = plain(z[i], u[i], g.get("temperature", 1.0), int(g.get("top_k", 0)),
                                   np.float32(g.get("top_p", 1.0)))
            # half a unit (vocab 2^-63) a token
            if want != idx[i] and 0 < room < V * V * 2.0 ** -63:
                continue
            assert idx[i] == want, (kw, i, room)
            assert abs(prob[i] - pr) <= 2.0 ** -20 * pr + V * 2.0 ** -62


def test_without_probabilities(gpu):
    """out_prob may be NULL, and so may every setting."""
    from rapidllm_amd import hip
    from rapidllm_amd.hip import DeviceBuffer, call

    z, u, _ = rows(23, 4, 5000)
    d, du, di = DeviceBuffer.from_numpy(z), DeviceBuffer.from_numpy(u), DeviceBuffer(16)
    t = DeviceBuffer.from_numpy(np.array([1, 0, 1, 0], np.float32))
    ws = DeviceBuffer(hip.lib().rl_hip_sample_workspace_bytes(4, 5000))
    call("rl_hip_sample_rows", F32, d.ptr, 5000, 4, 5000, t.ptr, None, None, None, du.ptr, di.ptr, None, ws.ptr,
         ws.nbytes, None)
    got = di.numpy(np.int32, (4,))
    assert got.tolist() == [plain(z[i], u[i], [1, 0, 1, 0][i])[0] for i in range(4)]


def test_runs_of_nan(gpu):
    """Whole stretches of a row are NaN: they count for nothing, also where maxima of stretches decide."""
    z, u, r = rows(29, 6, 60000)
    z[0, 512:1024] = np.nan
    z[1, :4096] = np.nan
    z[2, 10000:] = np.nan
    z[3, r.random(60000) < 0.9] = np.nan
    z[4, 1:] = np.nan
    for k in (1, 2, 5, 40):
        check(z, u, top_k=k)
        check(z, u, F16, top_k=k, top_p=0.9)
    check(z, u, top_p=0.95)
    check(z, u)
