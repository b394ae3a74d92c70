"""4-bit rows (include/ipx.h: ipx_mx4_*, storage 3, ipx_scores, ipx_lookup) against their definition in 64 bits.

Quantisation, dequantisation and lookup are exact, so they are compared for equality. A search of an mx4 index has to
return the bits of a bf16 index of the same values (both: the oracle's kernel-order scores of <fp32 query, stored value>).
Scores are compared with float64 within the error that the query's five-part split and fp32 sums can make (score_bound).
"""
import ctypes as C

import numpy as np
import pytest

import mx4_oracle as M
from conftest import gaussian
from oracle import oracle as O

pytestmark = pytest.mark.gpu
FLT_MAX = np.finfo(np.float32).max


@pytest.fixture(scope="module")
def R():
    from mural_amd.faiss_retriever import retriever
    from mural_amd import _lib
    assert _lib.lib().ipx_device_count() >= 1, "no HIP device visible: these operators have no CPU fallback"
    return retriever


@pytest.fixture(scope="module")
def mx4():
    from mural_amd import mx4
    return mx4


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def spread(seed, shape):
    """rows of very different scales, within and between rows"""
    r = np.random.default_rng(seed)
    return (r.standard_normal(shape) * np.exp(3 * r.standard_normal((shape[0], 1))) * np.exp(2 * r.standard_normal(shape))).astype(np.float32)


def index(R, X, storage="mx4", adds=1):
    ix = R.FlatIPIndex(X.shape[1], storage=storage)
    step = -(-X.shape[0] // adds) if X.shape[0] else 1
    for lo in range(0, X.shape[0], step):
        ix.add(X[lo:lo + step])
    assert ix.ntotal == X.shape[0]
    return ix


def assert_bits(D, I, Q, X, k):
    rD, rI = O.topk_total_order(O.scores_mfma_order(Q, X), k)
    assert np.array_equal(I, rI), f"ids differ at {np.argwhere(I != rI)[:3].tolist()}"
    assert np.array_equal(D.view(np.uint32), rD.view(np.uint32)), "score bits differ"


def same_values(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return np.array_equal(a, b, equal_nan=True) and np.array_equal(np.signbit(a) | np.isnan(a), np.signbit(b) | np.isnan(b))


# ---- quantisation ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,d", [(1, 1), (1, 768), (3, 31), (5, 32), (7, 33), (130, 100), (1000, 768), (33, 8191), (2, 65536)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_quantize_and_dequantize_equal_the_definition(torch, mx4, n, d, dtype):
    x = torch.from_numpy(np.clip(spread(n + d, (n, d)), -6e4, 6e4)).to(getattr(torch, dtype))
    codes, scales = mx4.quantize(x.cuda())
    rc, rs = M.quantize(x.double().numpy())
    assert np.array_equal(scales.cpu().numpy(), rs)
    assert np.array_equal(codes.cpu().numpy(), rc)
    ref = M.dequantize(rc, rs, d)
    assert same_values(mx4.dequantize(codes, scales, d).cpu(), ref)
    assert same_values(mx4.dequantize(codes, scales, d, dtype=torch.bfloat16).double().cpu(), ref)
    half = torch.from_numpy(ref).to(torch.float16)
    assert same_values(mx4.dequantize(codes, scales, d, dtype=torch.float16).cpu(), half)


def test_quantize_borders(torch, mx4):
    """ties, the clamp at 6, zeros of both signs, subnormals, the largest numbers, NaN and infinities"""
    f = np.float32
    half_steps = np.arange(-32, 33, dtype=f) / 8            # every tie of every step, both signs
    rows = [half_steps[:32], half_steps[32:64], half_steps[:32] * f(2.0 ** 100), half_steps[32:64] * f(2.0 ** -126),
            np.zeros(32, f), -np.zeros(32, f), np.full(32, np.finfo(f).tiny), np.arange(32).astype(f) * f(2.0 ** -149),
            np.full(32, FLT_MAX), np.full(32, 7.99, f), np.r_[f(np.nan), np.ones(31, f)], np.r_[np.ones(31, f), f(-np.inf)],
            np.r_[f(4.0), np.full(31, 1e-30, f)], np.r_[f(3.9999998), np.full(31, 0.125, f)]]
    x = np.stack(rows).astype(f)
    codes, scales = mx4.quantize(torch.from_numpy(x).cuda())
    rc, rs = M.quantize(x)
    assert np.array_equal(scales.cpu().numpy(), rs) and np.array_equal(codes.cpu().numpy(), rc)
    assert same_values(mx4.dequantize(codes, scales, 32).cpu(), M.dequantize(rc, rs, 32))


def test_every_scale_and_code_dequantizes(torch, mx4):
    codes = np.tile(np.array([2 * i | (2 * i + 1) << 4 for i in range(8)] * 2, np.uint8), (256, 1, 1))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    ref = M.dequantize(codes, scales, 32)
    out = mx4.dequantize(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), 32).cpu().numpy()
    ref32 = ref.astype(np.float32)                          # (scales 253 and 254 pass fp32's range: inf, as rounding gives)
    assert same_values(out, ref32)


@pytest.mark.parametrize("offset,width,d", [(0, 800, 768), (1, 801, 768), (3, 103, 100), (4, 40, 33), (0, 64, 1)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_quantize_strided_and_unaligned_views(torch, mx4, offset, width, d, dtype):
    base = torch.from_numpy(gaussian(offset + d, (50, width))).to(getattr(torch, dtype)).cuda()
    x = base[:, offset:offset + d]
    codes, scales = mx4.quantize(x)
    rc, rs = M.quantize(x.double().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), rc) and np.array_equal(scales.cpu().numpy(), rs)
    codes, scales = mx4.quantize(base.t()[:40])             # elements not adjacent: copied first
    rc, rs = M.quantize(base.t()[:40].double().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), rc) and np.array_equal(scales.cpu().numpy(), rs)


def test_numpy_rows_take_the_same_way(mx4):
    for x in (gaussian(5, (77, 100)), gaussian(6, (3, 768)).astype(np.float16), gaussian(7, (2, 5)).astype(np.float64)):
        codes, scales = mx4.quantize(x)
        rc, rs = M.quantize(x.astype(np.float32) if x.dtype == np.float64 else x)
        assert np.array_equal(codes, rc) and np.array_equal(scales, rs)
        assert same_values(mx4.dequantize(codes, scales, x.shape[1]), M.dequantize(rc, rs, x.shape[1]))
        assert mx4.dequantize(codes, scales, x.shape[1], dtype=np.float16).dtype == np.float16
    codes, scales = mx4.quantize(np.empty((0, 100), np.float32))
    assert codes.shape == (0, 4, 16) and mx4.dequantize(codes, scales, 100).shape == (0, 100)


# ---- search ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,d,nq,k,adds", [
    (4096, 768, 32, 1, 1), (4096, 768, 33, 100, 1), (5000, 768, 300, 100, 2),
    (20000, 100, 513, 100, 3), (9000, 17, 64, 512, 2), (9000, 48, 64, 1500, 1), (9000, 48, 130, 2048, 2),
    (777, 768, 1, 100, 1), (255, 16, 257, 5, 1), (257, 16, 256, 300, 1), (1, 8, 3, 4, 1), (33, 1, 2, 7, 33),
    (16384, 64, 5, 10, 1), (16385, 64, 5, 10, 2),
    (3000, 1000, 40, 50, 1), (3000, 1536, 129, 20, 1),     # fewer queries per block: longer vectors
    (2000, 4096, 70, 30, 1), (1500, 8192, 3, 20, 1),       # the query block goes through LDS in turns
])
def test_search_equals_the_exact_scores_of_the_stored_values(R, n, d, nq, k, adds):
    X, Q = gaussian(1234, (n, d)), gaussian(4321, (nq, d))
    ix = index(R, X, adds=adds)
    D, I = ix.search(Q, k)
    assert D.dtype == np.float32 and I.dtype == np.int64 and D.shape == (nq, k) == I.shape
    assert_bits(D, I, Q, M.rounded(X), k)


@pytest.mark.parametrize("n,d,nq,k", [(1, 8, 3, 4), (33, 1, 2, 7), (777, 768, 1, 100), (257, 16, 256, 128), (4000, 64, 40, 200),
                                      (4096, 33, 300, 10), (129, 8192, 2, 100)])
@pytest.mark.parametrize("candidates", [1, 300])
def test_short_indexes_through_the_scan(R, n, d, nq, k, candidates):
    """Short indexes are scored row by row; with a list length given they take the scan: the same answer."""
    X, Q = gaussian(1235, (n, d)), gaussian(4322, (nq, d))
    X[n // 2] = 0
    ix = index(R, X)
    D, I = ix.search(Q, k)
    assert_bits(D, I, Q, M.rounded(X), k)
    ix.set_param("bf16_candidates", candidates)
    D2, I2 = ix.search(Q, k)
    assert np.array_equal(I, I2) and np.array_equal(D.view(np.uint32), D2.view(np.uint32))


@pytest.mark.parametrize("n,d,nq,k", [(60000, 768, 64, 100), (120000, 96, 200, 1000), (50000, 768, 1, 10)])
def test_search_equals_a_bf16_index_of_the_same_values(R, n, d, nq, k):
    X, Q = gaussian(8, (n, d)), gaussian(9, (nq, d))
    ix = index(R, X)
    D, I = ix.search(Q, k)
    D2, I2 = index(R, M.rounded(X), "bf16").search(Q, k)
    assert np.array_equal(I, I2) and np.array_equal(D.view(np.uint32), D2.view(np.uint32))
    st = ix.last_bf16_stats()
    assert st["candidates"] >= k and st["exact_queries"] == 0


@pytest.mark.parametrize("n,d,nq,k", [(4095, 64, 300, 229), (4097, 40, 257, 2048), (8191, 33, 9, 100), (8192, 33, 9, 100),
                                      (8193, 320, 30, 229), (65537, 16, 3, 900), (3300, 512, 300, 2000), (2049, 100, 500, 3)])
@pytest.mark.parametrize("kind", ["plain", "shifted", "few numbers", "one score"])
def test_every_length_has_a_floor(R, n, d, nq, k, kind):
    """Floors from samples of every size, from scores that all lie on one side of zero, that are few, or equal."""
    X, Q = gaussian(n, (n, d)), gaussian(n + 1, (nq, d))
    if kind == "shifted":
        X[:, 0], Q[:, 0] = 40, np.where(np.arange(nq) % 2, 3, -3)
    elif kind == "few numbers":
        X[np.arange(n) % 41 != 7, 3 % d] = np.nan
    elif kind == "one score":
        X[:], Q[nq // 2] = X[0], 0
    ix = index(R, X)
    D, I = ix.search(Q, k)
    some = np.unique(np.r_[0, nq // 2, nq - 1, np.random.default_rng(1).integers(0, nq, 6)])
    assert_bits(D[some], I[some], Q[some], M.rounded(X), k)
    ix.set_param("bf16_candidates", 128)
    D2, I2 = ix.search(Q, k)
    assert np.array_equal(I, I2) and np.array_equal(D.view(np.uint32), D2.view(np.uint32))


def test_rows_in_groups_and_order_do_not_break_the_floor(R):
    """The floor comes from a sample: rows sorted by their score, the best ones in one place, or many equal ones must not
    change the answer."""
    d, n, k = 64, 40000, 50
    q = gaussian(1, (4, d))
    X = gaussian(2, (n, d))
    order = np.argsort(X @ q[0])
    for Y in (X[order], X[order[::-1]], np.r_[X[:20000] * 0.01, 5 * q[:1].repeat(300, 0), X[20300:] * 0.01].astype(np.float32),
              np.tile(X[:1], (n, 1)), np.tile(X[:7], (n // 7 + 1, 1))[:n]):
        Y = np.ascontiguousarray(Y)
        ix = index(R, Y)
        D, I = ix.search(q, k)
        assert_bits(D, I, q, M.rounded(Y), k)


def test_zero_nan_and_infinite_queries_and_rows(R):
    n, d, k = 20000, 96, 30
    X, Q = gaussian(3, (n, d)), gaussian(4, (9, d))
    X[5] = 0
    X[17, 3] = np.nan
    X[18001, 95] = np.inf
    Q[1] = 0
    Q[2, 5] = np.nan
    Q[4, 0] = np.inf
    Q[6] *= 1e-30                                           # squares vanish in fp32
    Q[7] = 0
    Q[7, 3] = 1e-38
    for m in (n, 3000):
        ix = index(R, X[:m])
        D, I = ix.search(Q, k)
        with np.errstate(all="ignore"):
            assert_bits(D, I, Q, M.rounded(X[:m]), k)
        assert not np.isin(I, [17, 18001]).any()
    e = R.FlatIPIndex(d, storage="mx4")
    D, I = e.search(Q, 3)
    assert (I == -1).all() and (D == -FLT_MAX).all()


def test_a_search_does_not_depend_on_its_batch(R):
    X, Q = gaussian(11, (30000, 200)), gaussian(12, (150, 200))
    ix = index(R, X)
    D, I = ix.search(Q, 40)
    for lo, hi in ((0, 1), (1, 33), (33, 97), (97, 150)):
        D2, I2 = ix.search(Q[lo:hi], 40)
        assert np.array_equal(I[lo:hi], I2) and np.array_equal(D[lo:hi], D2)
    for kc in (40, 64, 4096):                                # too short lists are repeated, long ones change nothing
        ix.set_param("bf16_candidates", kc)
        D2, I2 = ix.search(Q, 40)
        assert np.array_equal(I, I2) and np.array_equal(D, D2)


def test_aspect_queries_and_pooled_rows(R):
    """the other entry points of an index serve 4-bit rows too"""
    X = gaussian(21, (5000, 64))
    ix = index(R, X)
    emb, w = gaussian(22, (20, 3, 64)), np.abs(gaussian(23, (20, 3)))
    D, I = ix.search_aspect(emb, w, 10)
    q = np.zeros((20, 64), np.float32)
    ref = index(R, M.rounded(X), "bf16")
    D2, I2 = ref.search_aspect(emb, w, 10)
    assert np.array_equal(I, I2) and np.array_equal(D, D2)
    W, b, hid = gaussian(24, (3, 64)), gaussian(25, (3,)), gaussian(26, (40, 8, 64))
    ix.add_pooled(hid, W, b)
    rep, _ = ix.pool(hid, W, b)
    assert ix.ntotal == 5040
    assert np.array_equal(ix.lookup(np.arange(5000, 5040)), M.rounded(rep))


# ---- scores ------------------------------------------------------------------------------------------------------

def score_bound(Q, X):
    """|score - float64| at most: five E2M3 parts leave an element of q at most 2^-20 of its block's largest magnitude
    (each part at most 1/16 of what it rounds), and fewer than 5 x padded d additions round to 24 bits."""
    nq, d = Q.shape
    nb = -(-d // 32)
    pad = lambda a: np.pad(np.abs(a.astype(np.float64)), ((0, 0), (0, nb * 32 - d))).reshape(len(a), nb, 32)
    split = np.einsum("qb,nb->qn", pad(Q).max(2), pad(X).sum(2)) * 2.0 ** -20
    dpad = -(-d // 64) * 64
    return split + 5 * dpad * 2.0 ** -24 * (np.abs(Q.astype(np.float64)) @ np.abs(X.astype(np.float64)).T) + 1e-38


@pytest.mark.parametrize("nq,n,d,start,count", [
    (1, 1, 1, 0, 1), (1, 5000, 768, 0, 5000), (3, 999, 100, 0, 999), (33, 700, 100, 1, 699), (70, 333, 33, 37, 200),
    (129, 1000, 768, 63, 65), (64, 64, 64, 64, 0), (200, 300, 1536, 32, 255), (40, 130, 4096, 5, 100), (2, 70, 8192, 0, 70),
    (300, 2049, 260, 2048, 1)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_scores_are_fp32_products_with_the_stored_values(R, torch, nq, n, d, start, count, dtype):
    X = gaussian(31, (n, d))
    q = torch.from_numpy(gaussian(32, (nq, d))).to(getattr(torch, dtype))
    ix = index(R, X)
    Qd, Xr = q.double().numpy(), M.rounded(X)[start:start + count]
    ref = Qd @ Xr.astype(np.float64).T
    out = ix.scores(q.cuda(), start, count).cpu().numpy()
    assert out.shape == (nq, count)
    assert (np.abs(out - ref) <= score_bound(Qd, Xr)).all()
    if dtype != "bfloat16":
        host = ix.scores(q.numpy(), start, count)
        assert np.array_equal(host, out)
    if start == 0 and count == n:
        assert np.array_equal(ix.scores(q.cuda()).cpu().numpy(), out)


def test_scores_of_spread_queries(R, torch):
    """blocks whose elements differ by many orders of magnitude, rows too"""
    X, Q = spread(41, (500, 300)), spread(42, (40, 300))
    ix = index(R, X)
    Xr = M.rounded(X)
    out = ix.scores(torch.from_numpy(Q).cuda()).cpu().numpy()
    assert (np.abs(out - Q.astype(np.float64) @ Xr.astype(np.float64).T) <= score_bound(Q, Xr)).all()


@pytest.mark.parametrize("nq,n,d", [(1, 40, 32), (5, 999, 100), (100, 700, 768), (300, 130, 33), (64, 64, 2048), (3, 50, 8192)])
def test_scores_of_mx4_queries_are_exact(R, mx4, torch, nq, n, d):
    """Gaussian blocks: every product is a multiple of 2^-12 or so and every sum far below 2^12: exact in fp32."""
    X, Q = gaussian(51, (n, d)), gaussian(52, (nq, d))
    ix = index(R, X)
    ref = M.rounded(Q).astype(np.float64) @ M.rounded(X).astype(np.float64).T
    codes, scales = mx4.quantize(torch.from_numpy(Q).cuda())
    assert np.array_equal(ix.scores_mx4(codes, scales).cpu().numpy(), ref)
    assert np.array_equal(ix.scores_mx4(codes.cpu().numpy(), scales.cpu().numpy(), 1, n - 1), ref[:, 1:])
    if d % 32:                                              # codes behind the last element count for nothing
        codes[:, -1, -1] = 0x77
        assert np.array_equal(ix.scores_mx4(codes, scales).cpu().numpy(), ref)


def test_scores_of_queries_and_rows_that_are_not_finite(R, torch):
    X, Q = gaussian(61, (200, 100)), gaussian(62, (40, 100))
    X[3, 50] = np.nan
    X[7] = 0
    Q[1, 2], Q[5, 99], Q[9, 0], Q[33, 64] = np.inf, -np.inf, np.nan, np.inf
    Q[11] = 0
    Xr = M.rounded(X)
    with np.errstate(all="ignore"):
        ref = np.array([[np.sum(q.astype(np.float64) * x) for x in Xr.astype(np.float64)] for q in Q])
    out = index(R, X).scores(torch.from_numpy(Q).cuda()).cpu().numpy()
    fine = np.isfinite(ref)
    assert np.array_equal(np.isnan(out), np.isnan(ref)) and np.array_equal(out[~fine & ~np.isnan(ref)], ref[~fine & ~np.isnan(ref)])
    bound = score_bound(np.where(np.isfinite(Q), Q, 0), np.where(np.isfinite(Xr), Xr, 0))
    assert (np.abs(out[fine] - ref[fine]) <= bound[fine]).all()


# ---- lookup ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("storage", ["f32", "bf16scan", "bf16", "mx4"])
@pytest.mark.parametrize("d", [1, 8, 33, 100, 768])
def test_lookup_returns_the_stored_rows(R, torch, storage, d):
    X = gaussian(71, (700, d))
    ix = index(R, X, storage, adds=2)
    kept = {"mx4": M.rounded(X), "bf16": torch.from_numpy(X).bfloat16().float().numpy()}.get(storage, X)
    ids = np.random.default_rng(72).integers(0, 700, (9, 31))
    ids[0, :3] = -1
    ids[1] = 699
    s = gaussian(73, ids.shape)
    ref = np.where((ids >= 0)[..., None], kept[ids], 0).astype(np.float32)
    assert same_values(ix.lookup(ids), ref)
    assert same_values(ix.lookup(ids, s), np.where((ids >= 0)[..., None], ref * s[..., None], 0))
    ti, ts = torch.from_numpy(ids).cuda(), torch.from_numpy(s).cuda()
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        out = ix.lookup(ti, ts, dtype=dtype)
        want = torch.from_numpy(np.where((ids >= 0)[..., None], ref * s[..., None], 0).astype(np.float32)).to(dtype)
        assert out.dtype == dtype and same_values(out.double().cpu(), want.double())
    assert ix.lookup(ti[:0]).shape == (0, 31, d)
    ix.check()


def test_lookup_of_ids_outside_the_index(R, torch):
    from mural_amd import _lib
    X = gaussian(81, (100, 40))
    ix = index(R, X)
    ix.set_id_base(1000)
    kept = M.rounded(X)
    assert np.array_equal(ix.lookup(np.array([1000, 1099])), kept[[0, 99]])
    for bad in (0, 999, 1100, -2, 2 ** 62, -2 ** 63):
        with pytest.raises(_lib.IpxError):
            ix.lookup(np.array([1000, bad]))
        out = ix.lookup(torch.tensor([1001, bad], device="cuda"))
        assert np.array_equal(out.cpu().numpy(), np.stack([kept[1], np.zeros(40, np.float32)]))
        with pytest.raises(_lib.IpxError):
            ix.check()
        ix.check()                                          # reported once
    D, I = ix.search(gaussian(82, (3, 40)), 5)              # and a search is not disturbed by it
    assert (I >= 1000).all()


# ---- together ----------------------------------------------------------------------------------------------------

def test_quantize_ship_search_look_up_and_score(R, mx4, torch):
    """A 4-bit shard as a service uses it: rows quantised elsewhere are added, a query is searched, its passages are fetched
    and weighted into a second query, and the list is scored again."""
    X, Q = gaussian(91, (30000, 768)), gaussian(92, (8, 768))
    codes, scales = mx4.quantize(torch.from_numpy(X).cuda())
    ix = R.FlatIPIndex(768, storage="mx4")
    ix.add_mx4(codes[:10001], scales[:10001])
    ix.add_mx4(codes[10001:].cpu().numpy(), scales[10001:].cpu().numpy())
    assert ix.ntotal == 30000
    tq = torch.from_numpy(Q).cuda()
    D, I = ix.search(tq, 20)
    Xr = M.rounded(X)
    assert_bits(D.cpu().numpy(), I.cpu().numpy(), Q, Xr, 20)
    D1, I1 = index(R, X).search(Q, 20)                      # added as fp32 rows: the same index
    assert np.array_equal(I1, I.cpu().numpy()) and np.array_equal(D1, D.cpu().numpy())
    rows = ix.lookup(I, torch.softmax(D, 1))
    fed = tq + rows.sum(1)
    S = ix.scores(fed)
    assert S.shape == (8, 30000)
    D2, I2 = ix.search(fed, 20)
    bound = score_bound(fed.cpu().numpy(), Xr)
    assert (np.abs(S.cpu().numpy() - fed.cpu().numpy().astype(np.float64) @ Xr.astype(np.float64).T) <= bound).all()
    got = torch.gather(S, 1, I2).cpu().numpy()
    assert (np.abs(got - D2.cpu().numpy()) <= 2 * np.take_along_axis(bound, I2.cpu().numpy(), 1)).all()


def test_on_another_stream_and_in_a_graph(R, mx4, torch):
    """quantize, dequantize, scores and lookup neither synchronise nor clear memory by a fill of the runtime's: they replay
    from a captured graph with the results of eager calls."""
    X = torch.from_numpy(gaussian(95, (3000, 200))).cuda()
    ix = R.FlatIPIndex(200, storage="mx4")
    ix.add(X)
    q = torch.from_numpy(gaussian(96, (70, 200))).cuda()
    ids = torch.arange(0, 3000, 7, device="cuda")
    s = torch.rand(ids.shape[0], device="cuda")

    def work():
        codes, scales = mx4.quantize(q)
        return mx4.dequantize(codes, scales, 200), ix.scores(q), ix.scores_mx4(codes, scales, 5, 100), ix.lookup(ids, s)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(4):
        q.copy_(torch.from_numpy(gaussian(97 + i, (70, 200))))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        for a, b in zip(got, work()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("storage", ["mx4", "bf16", "f32"])
def test_a_graph_outlives_larger_calls_and_added_rows(R, mx4, torch, storage):
    """Buffers that a captured call uses are replaced, not freed, when a later call needs larger ones."""
    X = torch.from_numpy(gaussian(101, (1500, 96))).cuda()
    ix = R.FlatIPIndex(96, storage=storage)
    ix.add(X)
    q = torch.from_numpy(gaussian(102, (39, 96))).cuda()
    codes, scales = mx4.quantize(q)
    ids = torch.arange(1499, -1, -3, device="cuda")

    def work():
        if storage != "mx4":
            return (ix.lookup(ids),)
        return ix.scores(q, 0, 1500), ix.scores(q[:2], 0, 1500), ix.scores_mx4(codes, scales, 0, 1500), ix.lookup(ids)

    first = work()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for grow in range(3):
        for o in out:
            o.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, first))
        ix.add(torch.from_numpy(gaussian(103 + grow, (3000 << grow, 96))).cuda())
        if storage == "mx4":
            ix.scores(torch.from_numpy(gaussian(104, (2000, 96))).cuda())
        assert all(torch.equal(a, b) for a, b in zip(work(), first))


def test_scores_of_a_query_do_not_depend_on_the_others(R, torch):
    """Up to 32 queries are packed by the product kernel, more by a kernel before it: the same bits."""
    X, q = gaussian(105, (700, 300)), gaussian(106, (40, 300))
    q[1, 7], q[2, 299], q[3] = np.inf, np.nan, q[3] * np.float32(2.0 ** 100)
    ix = index(R, X)
    tq = torch.from_numpy(q).cuda()
    full = ix.scores(tq).cpu().numpy()
    for n in (1, 2, 3, 4, 5, 32, 33):
        for lo in (0, 1, 7):
            assert np.array_equal(ix.scores(tq[lo:lo + n]).cpu().numpy(), full[lo:lo + n], equal_nan=True)


@pytest.mark.parametrize("nq,n,start", [(1030, 65600, 0), (1100, 65536, 32), (1100, 65536, 64), (1100, 65537, 0)])
def test_scores_larger_than_the_caches(R, mx4, torch, nq, n, start):
    """Those of 256 MB and more are stored another way where their lines are whole: the bits of smaller calls."""
    ix = R.FlatIPIndex(200, storage="mx4")
    g = torch.Generator(device="cuda").manual_seed(nq + n)
    ix.add(torch.randn((n + 100, 200), generator=g, device="cuda"))
    q = torch.randn((nq, 200), generator=g, device="cuda")
    pair = mx4.quantize(q)
    for whole, part in ((ix.scores(q, start, n), ix.scores(q, start + 1000, 30000)),
                        (ix.scores_mx4(*pair, start, n), ix.scores_mx4(*pair, start + 1000, 30000))):
        assert torch.equal(whole[:, 1000:31000], part)
    few = mx4.quantize(q[-3:])
    assert torch.equal(whole[-3:], ix.scores_mx4(*few, start, n))
    q[5, 3] = float("inf")
    big = ix.scores(q, start, n)
    for lo, hi in ((0, 40), (40, 200)):
        assert torch.allclose(big[lo:hi], ix.scores(q[lo:hi], start, n), rtol=0, atol=0, equal_nan=True)


def test_scores_of_very_many_queries(R, mx4, torch):
    """More queries than one pass takes."""
    n = (1 << 18) + 70
    X = gaussian(107, (21, 40))
    ix = index(R, X)
    q = gaussian(108, (n, 40))
    tq = torch.from_numpy(q).cuda()
    Xr = M.dequantize(*M.quantize(X), 40)
    S = ix.scores(tq).cpu().numpy()
    assert (np.abs(S - q.astype(np.float64) @ Xr.astype(np.float64).T) <= score_bound(q, Xr)).all()
    codes, scales = mx4.quantize(tq)
    S = ix.scores_mx4(codes, scales, 1, 20)
    for lo in (0, (1 << 18) - 40, n - 70):
        assert torch.equal(S[lo:lo + 70], ix.scores_mx4(codes[lo:lo + 70], scales[lo:lo + 70], 1, 20))


def test_offsets_beyond_32_bits(R, mx4, torch):
    """An index of 4.6 GB and a score matrix of 5 GB: the last rows are found where they are."""
    d, n, step = 2048, 4300000, 430000
    g = torch.Generator(device="cuda").manual_seed(5)
    ix = R.FlatIPIndex(d, storage="mx4")
    for lo in range(0, n, step):
        x = torch.randn((step, d), generator=g, device="cuda", dtype=torch.float16)
        ix.add(x)
    tail = x[-300:].float()                        # rows n - 300 ..
    want = mx4.dequantize(*mx4.quantize(tail), d)
    ids = torch.arange(n - 300, n, device="cuda")
    assert torch.equal(ix.lookup(ids), want)
    D, I = ix.search(tail, 3)
    assert torch.equal(I[:, 0], ids)
    S = ix.scores(tail)
    Q, X = tail.cpu().numpy(), want.cpu().numpy()
    bound = score_bound(Q, X)
    ref = Q.astype(np.float64) @ X.astype(np.float64).T
    assert (np.abs(S[:, n - 300:].cpu().numpy() - ref) <= bound).all()
    assert torch.equal(S[:, n - 300:], ix.scores(tail, n - 300))
    assert torch.equal(S[:, 77:99], ix.scores(tail, 77, 22))
    assert (np.abs(D[:, 0].cpu().numpy() - np.diag(ref)) <= np.diag(bound)).all()


def test_storage_rules(R, mx4):
    from mural_amd import _lib
    ix = R.FlatIPIndex(64, storage="mx4")
    ix.add(gaussian(1, (10, 64)))
    for name, value in (("storage", 0), ("f32_scan", 1)):
        with pytest.raises(_lib.IpxError):
            ix.set_param(name, value)
    with pytest.raises(_lib.IpxError):
        ix.search(gaussian(2, (1, 64)), 2049)
    q = gaussian(2, (2, 64))
    for start, n in ((-1, 2), (0, 11), (10, 1), (11, 0), (0, -1), (3, 2 ** 62)):
        with pytest.raises((_lib.IpxError, ValueError)):
            ix.scores(q, start, n) if abs(n) < 100 else _lib.check(_lib.lib().ipx_scores(ix._h, C.c_void_p(q.ctypes.data), 0, 2, start, n, C.c_void_p(q.ctypes.data), 0, None))
    assert ix.scores(q, 10, 0).shape == (2, 0) and ix.scores(q[:0]).shape == (0, 10)
    with pytest.raises(AssertionError):
        ix.scores(gaussian(1, (2, 63)))
    with pytest.raises(AssertionError):
        ix.add_mx4(np.zeros((3, 3, 16), np.uint8), np.zeros((3, 3), np.uint8))
    with pytest.raises(_lib.IpxError):
        R.FlatIPIndex(8193, storage="mx4")
    plain = R.FlatIPIndex(64)
    plain.add(gaussian(1, (10, 64)))
    codes, scales = mx4.quantize(q)
    for call in (lambda: plain.scores(q), lambda: plain.scores_mx4(codes, scales), lambda: plain.add_mx4(codes, scales)):
        with pytest.raises(_lib.IpxError):
            call()


def test_the_command_serves_4_bit_rows(R, tmp_path, monkeypatch):
    """IPX_STORAGE=mx4: the command's ranking is the search of the 4-bit values."""
    import pickle
    from argparse import Namespace
    from mural_amd.faiss_retriever import BaseFaissIPRetriever
    from mural_amd.faiss_retriever.__main__ import search_queries
    monkeypatch.setenv("IPX_STORAGE", "mx4")
    X, Q = gaussian(101, (2000, 96)), gaussian(102, (20, 96))
    r = BaseFaissIPRetriever(X)
    r.add(X)
    scores, ids = search_queries(r, Q, [f"d{i}" for i in range(2000)], Namespace(batch_size=7, depth=10, quiet=True))
    rD, rI = O.topk_total_order(O.scores_mfma_order(Q, M.rounded(X)), 10)
    assert np.array_equal(scores, rD) and ids.tolist() == [[f"d{i}" for i in row] for row in rI]
