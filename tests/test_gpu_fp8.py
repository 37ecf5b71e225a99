"""GPU parity of the 8-bit block-scaled operators: quantisers (codes equal to the exact rule's), the product, the routed experts, against 64-bit forms."""
import numpy as np
import pytest

import fp8_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    import eke_hive_b200 as E
    return E


def gen(seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows(M, K, seed, ld=None):
    """bf16 rows whose blocks have very different sizes, among them blocks of zeros."""
    import torch
    g = gen(seed)
    x = torch.randn(M, ld or K, device="cuda", generator=g)
    x = x * torch.exp2(torch.randint(-12, 12, (M, -(-(ld or K) // 128)), device="cuda", generator=g).float()).repeat_interleave(128, 1)[:, :(ld or K)]
    x[torch.rand(x.shape, device="cuda", generator=g) < 0.05] = 0.0
    x = x.to(torch.bfloat16)
    x[M // 2, :128] = 0.0
    return x[:, :K]


def matrix(N, K, seed):
    import torch
    g = gen(seed)
    q = (torch.randn(N, K, device="cuda", generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = (torch.rand(R.up(N), R.up(K), device="cuda", generator=g) + 0.5) * 2e-4
    return q, s


def record(E, H, I, seed, at=0):
    """A record in a buffer of its own, `at` bytes (a multiple of 16) behind a 4096-byte boundary, and its parts in 64 bits."""
    import torch
    mats = [matrix(I, H, seed), matrix(I, H, seed + 1), matrix(H, I, seed + 2)]
    buf = torch.zeros(E.Fp8RecLayout(H, I).total + at, dtype=torch.uint8, device="cuda")
    return E.fp8_record(H, I, *mats, out=buf[at:]), [(q.double(), s.double()) for q, s in mats]


# ---------------------------------------------------------------------------------------------------- quantisers
@pytest.mark.parametrize("M,K,ld", [(1, 128, None), (1, 16, None), (3, 2048, None), (67, 1552, None), (5, 400, 408), (9, 272, 275), (513, 7168, None), (2, 17408, None)])
def test_quant_rows_is_exact(E, M, K, ld):
    import torch
    x = rows(M, K, M + K, ld)
    q, s = E.fp8_quant_rows(x)
    q0, s0 = R.quant_rows(x.double())
    assert torch.equal(R.codes_to_f64(q), q0)
    assert torch.equal(s.double(), s0)


def test_quant_rows_every_bf16_quotient_border(E):
    """All pairs (amax, v) of bf16 mantissas, signs and a few exponents: ties between codes are seen as ties."""
    import torch
    man = 1.0 + torch.arange(128, device="cuda").float() / 128
    x = torch.zeros(128, 8, 128, device="cuda")
    for j, e in enumerate((0, -1, -2, -3, -5, -8, -10, -14)):
        x[:, j, :] = man[None, :] * 2.0 ** e * torch.where(torch.arange(128, device="cuda") % 2 == 0, 1.0, -1.0)
    x = torch.where(x.abs() > man[:, None, None], 0.5 * x, x)
    x[:, :, 0] = man[:, None]
    for scale in (1.0, 2.0 ** 100, 2.0 ** -100, 2.0 ** 126, 2.0 ** -120):
        xb = (x.reshape(128, 1024) * scale).to(torch.bfloat16)
        q, s = E.fp8_quant_rows(xb)
        q0, s0 = R.quant_rows(xb.double())
        assert torch.equal(R.codes_to_f64(q), q0), scale
        assert torch.equal(s.double(), s0), scale


def test_quant_rows_non_finite_blocks(E):
    import torch
    x = torch.randn(4, 512, device="cuda").to(torch.bfloat16)
    x[0, 5] = float("nan"); x[1, 200] = float("inf"); x[2, 500] = -float("inf")
    q, s = E.fp8_quant_rows(x)
    nan = torch.isnan(s)
    assert nan.nonzero().tolist() == [[0, 0], [1, 1], [3, 2]]
    assert (q[0, :128] == 0).all() and (q[1, 128:256] == 0).all() and (q[2, 384:] == 0).all()
    ok = E.fp8_quant_rows(x[3:4])
    assert torch.equal(q[3], ok[0][0]) and torch.equal(s[:, 3], ok[1][:, 0])
    W = matrix(130, 512, 3)
    y = E.fp8_gemm(E.GMat(E.FMT_FP8_B128, 130, 512, *W), q, s)
    assert torch.isnan(y[:3]).all() and torch.isfinite(y[3]).all()


def test_quant_rows_strides_and_rows_behind_the_last(E):
    import torch
    x = rows(5, 320, 1, 333)
    q = torch.full((8, 400), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((3, 9), -7.0, device="cuda")
    E.fp8_quant_rows(x, q=q[:5, :320], s=s[:, :5])
    q0, s0 = E.fp8_quant_rows(x.contiguous())
    assert torch.equal(q[:5, :320], q0) and torch.equal(s[:, :5], s0)
    assert (q[5:] == 0x55).all() and (q[:, 320:] == 0x55).all() and (s[:, 5:] == -7).all()


@pytest.mark.parametrize("N,K,dt", [(128, 128, "float32"), (1, 16, "float32"), (300, 1552, "float32"), (2111, 528, "bfloat16"), (129, 2048, "bfloat16"), (5120, 272, "float32")])
def test_quantize_is_exact(E, N, K, dt):
    import torch
    w = (torch.randn(N, K, device="cuda", generator=gen(N)) * 0.02).to(getattr(torch, dt))
    if N > 200:
        w[:128, :128] = 0.0
    q, s = E.fp8_quantize(w)
    q0, s0 = R.quant_blocks(w)
    assert torch.equal(R.codes_to_f64(q), q0)
    assert torch.equal(s.double(), s0)


# ---------------------------------------------------------------------------------------------------- the product
GEMM = [(1, 128, 128), (1, 1, 16), (1, 5120, 2048), (2, 300, 400), (7, 4100, 1552), (13, 256, 7168), (16, 384, 640), (17, 130, 272), (33, 1000, 1024), (64, 512, 512), (65, 257, 2064),
        (127, 640, 384), (128, 256, 256), (129, 255, 144), (200, 1500, 1000 // 16 * 16), (333, 513, 2048), (600, 260, 4096), (1030, 777, 528)]


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,N,K", GEMM)
def test_gemm(E, M, N, K, dt):
    import torch
    q, s = matrix(N, K, N + K)
    xq, xs = E.fp8_quant_rows(rows(M, K, M))
    y = E.fp8_gemm(E.GMat(E.FMT_FP8_B128, N, K, q, s), xq, xs, out_dtype=getattr(torch, dt))
    y0, a = R.gemm(R.codes_to_f64(xq), xs.double(), q.double(), s.double())
    tol = R.sum_bound(K) * a
    tol = tol + R.HALF[y.dtype] * (y0.abs() + tol)
    bad = (y.double() - y0).abs() > tol
    assert not bad.any(), (bad.sum().item(), bad.nonzero()[:4].tolist(), ((y.double() - y0).abs() / (a + 1e-300)).max().item())


# items split among two and four CTAs, behind whole rounds and without any, over a K that does not divide; pairs' items cut through the workspace
@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,N,K", [(33, 300, 4096), (70, 1100, 2192), (128, 5000, 4112), (300, 2900, 2320), (150, 20000, 2304), (300, 15000, 2176), (512, 1281, 9216)])
def test_gemm_split_items(E, M, N, K, dt):
    test_gemm(E, M, N, K, dt)


# few weight tiles and a long K: the sums stay in the workspace that the library asks for
@pytest.mark.parametrize("K", [13312, 16384, 20480])
@pytest.mark.parametrize("N", [64, 256, 1024])
@pytest.mark.parametrize("M", [5, 30, 33, 64, 128, 140])
def test_gemm_long_k_stays_in_its_workspace(E, M, N, K):
    import torch
    q, s = matrix(N, K, N + K)
    xq, xs = E.fp8_quant_rows(rows(M, K, M))
    room = E.fp8_gemm_ws_bytes(M, N, K)
    buf = torch.full((room + (64 << 20),), 0x5a, dtype=torch.uint8, device="cuda")
    y = E.fp8_gemm(E.GMat(E.FMT_FP8_B128, N, K, q, s), xq, xs, out_dtype=torch.float32, ws=buf[:room])
    assert (buf[room:] == 0x5a).all()
    y0, a = R.gemm(R.codes_to_f64(xq), xs.double(), q.double(), s.double())
    tol = R.sum_bound(K) * a
    assert ((y.double() - y0).abs() <= tol + R.HALF[torch.float32] * (y0.abs() + tol)).all()
    E.context().check_device()


def test_gemm_strides_and_what_lies_around(E):
    import torch
    M, N, K = 37, 201, 336
    q, s = matrix(N, K, 5)
    W = E.GMat(E.FMT_FP8_B128, N, K, q, s)
    xq, xs = E.fp8_quant_rows(rows(M, K, 6))
    for dt in (torch.bfloat16, torch.float32):
        ref = E.fp8_gemm(W, xq, xs, out_dtype=dt)
        xq2 = torch.full((M + 3, 512), 0x7f, dtype=torch.uint8, device="cuda")          # NaN codes around the rows
        xs2 = torch.full((3, M + 5), float("nan"), device="cuda")
        y = torch.full((M + 2, 233), -7.0, dtype=dt, device="cuda")
        xq2[:M, :K] = xq; xs2[:, :M] = xs
        E.fp8_gemm(W, xq2[:M, :K], xs2[:, :M], y=y[:M, :N])
        assert torch.equal(y[:M, :N], ref)
        assert (y[M:] == -7).all() and (y[:, N:] == -7).all()


def test_gemm_nan_codes_and_scales_stay_in_their_row_and_column(E):
    import torch
    M, N, K = 40, 300, 512
    q, s = matrix(N, K, 5)
    xq, xs = E.fp8_quant_rows(rows(M, K, 6))
    ref = E.fp8_gemm(E.GMat(E.FMT_FP8_B128, N, K, q, s), xq, xs)
    xq2, q2 = xq.clone(), q.clone()
    xq2[3, 100] = 0x7f
    q2.view(torch.uint8)[200, 7] = 0xff
    y = E.fp8_gemm(E.GMat(E.FMT_FP8_B128, N, K, q2, s), xq2, xs)
    nan = torch.isnan(y)
    assert nan[3].all() and nan[:, 200].all() and nan.sum() == N + M - 1
    assert torch.equal(y[~nan], ref[~nan])


@pytest.mark.parametrize("N,K", [(5120, 2048), (640, 7168)])
def test_gemm_twice_and_row_by_row(E, N, K):
    """The same call gives the same bits."""
    import torch
    q, s = matrix(N, K, 9)
    W = E.GMat(E.FMT_FP8_B128, N, K, q, s)
    for M in (1, 5, 16, 40, 150):
        xq, xs = E.fp8_quant_rows(rows(M, K, M))
        a = E.fp8_gemm(W, xq, xs, out_dtype=torch.float32)
        for _ in range(3):
            assert torch.equal(a, E.fp8_gemm(W, xq, xs, out_dtype=torch.float32))


def test_gemm_refusals(E):
    import torch
    q, s = matrix(64, 256, 1)
    W = E.GMat(E.FMT_FP8_B128, 64, 256, q, s)
    xq, xs = E.fp8_quant_rows(rows(4, 256, 2))
    with pytest.raises(E.HbError):
        E.fp8_gemm(E.GMat(E.FMT_NVFP4, 64, 256, q, s), xq, xs)
    with pytest.raises(E.HbError):
        E.fp8_gemm(E.GMat(E.FMT_FP8_B128, 64, 248, q, s), xq, xs)
    with pytest.raises(E.HbError):
        E.fp8_gemm(W, xq[:, 8:], xs)                                                    # not 16-byte aligned
    with pytest.raises(E.HbError):
        E.fp8_gemm(W, xq, xs, y=torch.empty(4, 60, device="cuda"))
    with pytest.raises(E.HbError):
        E.fp8_gemm(W, xq, xs[:, :2].contiguous())                                       # fewer scales than rows
    with pytest.raises(E.HbError):
        E.fp8_gemm(W, xq, xs, ws=torch.empty(1024, dtype=torch.uint8, device="cuda")[8:])
    with pytest.raises(E.HbError):
        E.dense_gemv(W, rows(1, 256, 3), ws=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))   # the bf16-activation GEMV has no such format
    with pytest.raises(E.HbError):
        E.fp8_quant_rows(rows(2, 264, 3))
    assert E.fp8_gemm(W, xq[:0], xs[:, :0]).shape == (0, 64)
    assert E.fp8_quant_rows(rows(4, 256, 2)[:0])[0].shape == (0, 256)


# ---------------------------------------------------------------------------------------------------- routed experts
def routing(M, K, Ex, seed, hot=None):
    import torch
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.permutation(Ex)[:K] for _ in range(M)]).astype(np.int32)
    if hot is not None:
        ids[:, 0] = hot
        ids[:, 1:][ids[:, 1:] == hot] = (hot + 1) % Ex
    return torch.from_numpy(ids).cuda(), torch.from_numpy(rng.uniform(0.05, 0.6, (M, K)).astype(np.float32)).cuda()


def moe_check(E, M, H, I, Ex, K, seed, limit=0.0, hot=None, missing=(), shared=True, gate=True, edit=None):
    import torch
    recs = [record(E, H, I, 10 * e + seed, at=16 * (e % 7)) for e in range(Ex)]
    tab = torch.tensor([0 if e in missing else r[0].data_ptr() for e, r in enumerate(recs)], dtype=torch.int64, device="cuda")
    ref = [None if e in missing else r[1] for e, r in enumerate(recs)]
    x = (torch.randn(M, H, device="cuda", generator=gen(seed)) * 2).to(torch.bfloat16)
    ids, w = routing(M, K, Ex, seed, hot)
    if edit:
        edit(ids)
    sh = (torch.randn(M, H, device="cuda", generator=gen(seed + 1)) * 0.3).to(torch.bfloat16)
    lg = torch.randn(M, 3, device="cuda", generator=gen(seed + 2))
    o0, tol, mag = R.moe(ids, w, ref, x, limit)
    out = E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, limit=limit, out_dtype=torch.float32)
    err = (out.double() - o0).abs()
    assert (err <= tol + 1e-30).all(), ((err / (tol + 1e-30)).max().item(), (err > tol).sum().item())
    # tol adds up every rounding at its worst.  Over all outputs they do not conspire: d's rounding is off by 2^-8 of it at most, a code of y that falls the
    # other way (one in 2^16, where g and u are off by 2^-20) by 2^-3 of a value, 2^-11 of d; twice the first covers both
    assert err.norm() <= 2.0 ** -7 * mag.norm()
    s0, stol, _ = R.moe(ids, w, ref, x, limit, sh if shared else None, lg[:, 1] if gate else None)
    out = E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, shared=sh if shared else None, lg=lg if shared and gate else None, col=1, limit=limit)
    stol = stol + R.HALF[torch.bfloat16] * (s0.abs() + stol)
    err = (out.double() - s0).abs()
    assert (err <= stol + 1e-30).all(), (err / (stol + 1e-30)).max().item()
    assert torch.equal(out, E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, shared=sh if shared else None, lg=lg if shared and gate else None, col=1, limit=limit))
    return out


@pytest.mark.parametrize("M,H,I,Ex,K", [(1, 128, 128, 1, 1), (1, 2048, 512, 12, 10), (2, 256, 384, 6, 3), (5, 640, 256, 4, 4), (16, 2048, 512, 32, 10), (17, 512, 128, 3, 2), (40, 384, 640, 5, 4),
                                        (64, 1024, 256, 8, 8), (65, 256, 256, 2, 1), (130, 512, 384, 9, 4), (300, 256, 512, 2, 2), (700, 384, 256, 16, 5)])
def test_moe(E, M, H, I, Ex, K):
    moe_check(E, M, H, I, Ex, K, M + H)


# (pairs, pairs an expert): a list of 32 and one more; the longest that the kernels order for themselves and one more; experts just at 8 and 24 pairs on
# average and above; more experts than rows; the most experts and picks a call may have
@pytest.mark.parametrize("M,Ex,K", [(8, 4, 4), (11, 4, 3), (256, 160, 4), (205, 150, 5), (16, 4, 2), (17, 4, 2), (48, 4, 2), (49, 4, 2), (600, 80, 3), (3, 1024, 32), (40, 1024, 32)])
def test_moe_lists_of_pairs(E, M, Ex, K):
    """Every way the pairs are put in order and cut into tiles, over few different records."""
    import torch
    H, I, R0 = 256, 128, 6
    recs = [record(E, H, I, 10 * e + M) for e in range(R0)]
    tab = torch.tensor([0 if e % 13 == 5 else recs[e % R0][0].data_ptr() for e in range(Ex)], dtype=torch.int64, device="cuda")
    ids, w = routing(M, K, Ex, M)
    ids[M // 2, 0] = Ex; ids[0, K - 1] = -5
    x = (torch.randn(M, H, device="cuda", generator=gen(M)) * 2).to(torch.bfloat16)
    # of the same record: the reference's expert
    at = torch.where((ids >= 0) & (ids < Ex) & (ids % 13 != 5), ids % R0, -1)
    o0, tol = torch.zeros(M, H, dtype=torch.float64, device="cuda"), torch.zeros(M, H, dtype=torch.float64, device="cuda")
    for k in range(K):                                                                  # pair by pair: a row may have a record more than once
        o, t, _ = R.moe(at[:, k:k + 1], w[:, k:k + 1], [r[1] for r in recs], x)
        o0 += o; tol += t
    tol += 2.0 ** -23 * K * K * o0.abs() + 2.0 ** -23 * K * tol                         # the sum over the picks: an addition each, of sums no larger than all together
    out = E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, out_dtype=torch.float32)
    big = torch.zeros_like(o0)
    for k in range(K):
        o, _, _ = R.moe(at[:, k:k + 1], w[:, k:k + 1], [r[1] for r in recs], x)
        big += o.abs()
    assert ((out.double() - o0).abs() <= tol + 2.0 ** -23 * K * big + 1e-30).all()
    assert torch.equal(out, E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, out_dtype=torch.float32))


# experts whose runs take several tiles, of which some items are cut and others are not: tiles of 128 rows behind a round of whole items, tiles of 32 rows of more
# pairs than the kernels order for themselves, and a list that several CTAs put in order
@pytest.mark.parametrize("M,H,I,Ex,K,hot", [(1000, 2304, 1280, 4, 2, None), (750, 1024, 256, 80, 2, None), (750, 2304, 256, 80, 2, 3), (3000, 2304, 512, 6, 4, 1), (1200, 640, 384, 600, 12, None)])
def test_moe_long_lists_give_the_same_bits_every_time(E, M, H, I, Ex, K, hot):
    import torch
    R0 = min(Ex, 6)
    recs = [record(E, H, I, 10 * e + M)[0] for e in range(R0)]
    tab = torch.tensor([recs[e % R0].data_ptr() for e in range(Ex)], dtype=torch.int64, device="cuda")
    ids, w = routing(M, K, Ex, M, hot)
    x = (torch.randn(M, H, device="cuda", generator=gen(M)) * 2).to(torch.bfloat16)
    ref = E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, out_dtype=torch.float32)
    for _ in range(10):
        assert torch.equal(ref, E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, out_dtype=torch.float32))
    E.context().check_device()


def test_few_ctas_and_many(E):
    """Contexts that may use fewer CTAs cut the items elsewhere: the results stay within fp32 summation order, cut items or not."""
    import torch
    for M, N, K in ((1, 1000, 2048), (20, 640, 1024), (50, 500, 2048), (100, 700, 1536), (300, 1100, 1024)):
        q, s = matrix(N, K, N)
        W = E.GMat(E.FMT_FP8_B128, N, K, q, s)
        xq, xs = E.fp8_quant_rows(rows(M, K, M))
        y0, a = R.gemm(R.codes_to_f64(xq), xs.double(), q.double(), s.double())
        tol = R.sum_bound(K) * a
        tol = tol + R.HALF[torch.float32] * (y0.abs() + tol)
        for n in (1, 2, 3, 7, 64, 147):
            ctx = E.Context(max_ctas=n)
            y = E.fp8_gemm(W, xq, xs, out_dtype=torch.float32, ctx=ctx)
            assert ((y.double() - y0).abs() <= tol).all(), (M, n)
            ctx.check_device()
    H, I, Ex, Kk, M = 512, 256, 5, 3, 70
    recs = [record(E, H, I, 10 * e) for e in range(Ex)]
    tab = E.rec_table([r[0] for r in recs])
    x = torch.randn(M, H, device="cuda", generator=gen(7)).to(torch.bfloat16)
    for m in (1, 12, M):
        ids, w = routing(m, Kk, Ex, m)
        o0, tol, _ = R.moe(ids, w, [r[1] for r in recs], x[:m])
        for n in (1, 5, 40):
            ctx = E.Context(max_ctas=n)
            out = E.moe_fp8(ids, w, tab, 0, Ex, x[:m], H, I, out_dtype=torch.float32, ctx=ctx)
            assert ((out.double() - o0).abs() <= tol).all(), (m, n)
            ctx.check_device()


def test_two_contexts_at_once(E):
    """Calls on two streams, a context each: counters and workspaces are their own."""
    import torch
    N, K, H, I, Ex = 5120, 4096, 512, 256, 8
    W = [E.GMat(E.FMT_FP8_B128, N, K, *matrix(N, K, i)) for i in range(2)]
    recs = [record(E, H, I, 10 * e)[0] for e in range(Ex)]                              # (the table holds addresses: the records have to stay)
    tab = E.rec_table(recs)
    jobs = []
    for i, M in enumerate((5, 9, 300, 520)):
        x = rows(M, K, i)
        xq, xs = E.fp8_quant_rows(x)
        xe = torch.randn(M, H, device="cuda", generator=gen(i)).to(torch.bfloat16)
        jobs.append((W[i % 2], xq, xs, *routing(M, 2, Ex, i), xe))

    def run(j, ctx=None):
        w, xq, xs, ids, wt, xe = j
        return E.fp8_gemm(w, xq, xs, ctx=ctx), E.moe_fp8(ids, wt, tab, 0, Ex, xe, H, I, ctx=ctx)
    ref = [run(j) for j in jobs]
    streams, ctxs = [torch.cuda.Stream() for _ in range(2)], [E.Context() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for i in range(len(jobs)):
            for s in range(2):
                with torch.cuda.stream(streams[s]):
                    got.append(((i + s) % len(jobs), run(jobs[(i + s) % len(jobs)], ctxs[s])))
        torch.cuda.synchronize()
        for i, g in got:
            assert all(torch.equal(a, b) for a, b in zip(g, ref[i])), i
    for c in ctxs:
        c.check_device()


def test_gemm_matrix_beyond_32_bits(E):
    """Rows of a weight, and rows of x, more than 2^32 bytes from their first."""
    import torch
    M, N, K = 3, 300000, 16384
    q = torch.zeros(N, K, dtype=torch.uint8, device="cuda")
    s = torch.ones(R.up(N), R.up(K), device="cuda")
    part, _ = matrix(256, K, 1)
    q[-256:] = part.view(torch.uint8)
    xq, xs = E.fp8_quant_rows(rows(M, K, M))
    y = E.fp8_gemm(E.GMat(E.FMT_FP8_B128, N, K, q, s), xq, xs, out_dtype=torch.float32)
    y0, a = R.gemm(R.codes_to_f64(xq), xs.double(), part.double(), s[:2].double())
    assert (y[:, :-256] == 0).all()
    assert ((y[:, -256:].double() - y0).abs() <= R.sum_bound(K) * a + R.HALF[torch.float32] * (y0.abs() + R.sum_bound(K) * a)).all()
    del y
    # the same memory as rows of x: the last 300 of them, and all in one call
    part2, s2 = matrix(130, K, 2)
    xs = torch.ones(R.up(K), N, device="cuda")
    y = E.fp8_gemm(E.GMat(E.FMT_FP8_B128, 130, K, part2, s2), q, xs, out_dtype=torch.float32)
    y0, a = R.gemm(part.double(), torch.ones(R.up(K), 256, dtype=torch.float64, device="cuda"), part2.double(), s2.double())
    assert (y[:-256] == 0).all()
    assert ((y[-256:].double() - y0).abs() <= R.sum_bound(K) * a + R.HALF[torch.float32] * (y0.abs() + R.sum_bound(K) * a)).all()


def exact_experts(E, M, Ex, seed):
    """Experts whose y is known to the last bit: x holds e4m3 values up to 448 (scale 1), every gate is 56 (silu leaves it), up adds a few exact products, w2 is
    the unit matrix.  Returns (x, ids, w, table, its records, y fp32 [M, I])."""
    import torch
    H = I = 256
    g = gen(seed)
    unit = lambda n: torch.ones(n // 128, n // 128, device="cuda")
    x = torch.zeros(M, H, device="cuda")
    x[:, 0] = 448.0
    x[:, 1:9] = (torch.rand(M, 8, device="cuda", generator=g) * 400 + 40).to(torch.float8_e4m3fn).float() * torch.where(torch.rand(M, 8, device="cuda", generator=g) < 0.5, 1.0, -1.0)
    recs, ups = [], []
    for e in range(Ex):
        gate, up, down = (torch.zeros(n, k, device="cuda") for n, k in ((I, H), (I, H), (H, I)))
        gate[:, 0] = 1.0
        up[:, 1:9] = (torch.randn(I, 8, device="cuda", generator=g) * 2).to(torch.float8_e4m3fn).float()
        up[:, 1:9] = torch.where(up[:, 1:9].abs() < 0.25, 0.25, up[:, 1:9])                # (a sum of eight products then fits into 24 bits)
        down[torch.arange(H), torch.arange(I)] = 1.0
        f8 = [m.to(torch.float8_e4m3fn) for m in (gate, up, down)]
        recs.append(E.fp8_record(H, I, (f8[0], unit(I) * 0.125), (f8[1], unit(I) * 2.0 ** -9), (f8[2], unit(I))))
        ups.append(up)
    ids = torch.randint(0, Ex, (M, 1), device="cuda", generator=g, dtype=torch.int32)
    y = torch.stack([(x[m].double() @ ups[int(ids[m, 0])].double().T) * 2.0 ** -9 for m in range(M)])
    assert (y == y.float().double()).all()                                               # up's sums are fp32 values
    return x.to(torch.bfloat16), ids, torch.ones(M, 1, device="cuda"), E.rec_table(recs), recs, 56.0 * y.float()


@pytest.mark.parametrize("M,Ex", [(1, 4), (9, 4), (40, 4), (90, 4), (150, 4), (1100, 150), (1100, 60)])
def test_moe_sums_fp32_values(E, M, Ex):
    """A pair's result is no bf16 number on its way into the sum: each is a code of y times its block's scale, to fp32 precision."""
    import torch
    x, ids, w, tab, _recs, y = exact_experts(E, M, Ex, M)
    out = E.moe_fp8(ids, w, tab, 0, Ex, x, 256, 256, out_dtype=torch.float32).double()
    s = (y.abs().view(M, 2, 128).amax(2).double() / 448.0).float().double().repeat_interleave(128, 1)
    v = out / s
    assert ((v - y.double() / s).abs() <= 2.0 ** -4 * (y.double() / s).abs() + 2.0 ** -10 + 1e-4).all()      # its own code, or off a border the other one
    assert ((v - R.nearest_e4m3(v.clamp(-448, 448))).abs() <= 2.0 ** -22 * v.abs()).all()                   # the scale's product and the sum's rounding: half a step each


@pytest.mark.parametrize("M,Ex", [(1, 1), (8, 1), (30, 4), (90, 4), (600, 4), (1100, 60)])
def test_moe_quantises_y_by_the_rows_rule(E, M, Ex):
    """y · 448 / amax is a border between two codes, exactly, in every row and for every size of y: the code is the even one."""
    import torch
    H = I = 128
    mids = [m * 2.0 ** p for p in (-1, 0, 1, 2, 3) for m in range(17, 32, 2) if m * 2.0 ** p < 440]
    gate, up, down = (torch.zeros(n, k, device="cuda") for n, k in ((I, H), (I, H), (H, I)))
    gate[:, 0] = 1.0
    down[torch.arange(H), torch.arange(I)] = 1.0
    for i, m in enumerate([448.0] + mids):                                               # up's row i is m times a row's number: m in two codes, for a number in three values
        c = float(R.nearest_e4m3(torch.tensor([m * (1 - 2.0 ** -6)], dtype=torch.float64)))
        up[i, 1:4], up[i, 4:7] = c, m - c
    assert (up.to(torch.float8_e4m3fn).float() == up).all() and ((up[1:len(mids) + 1, 1] + up[1:len(mids) + 1, 4]).cpu() == torch.tensor(mids)).all()
    one = torch.ones(1, 1, device="cuda")
    f8 = [m.to(torch.float8_e4m3fn) for m in (gate, up, down)]
    rec = E.fp8_record(H, I, (f8[0], one * 0.125), (f8[1], one * 2.0 ** -9), (f8[2], one))
    x = torch.zeros(M, H, dtype=torch.float64, device="cuda")
    x[:, 0] = 448.0
    number = (torch.arange(M, device="cuda", dtype=torch.float64) * 7 + 3) % 700 + 1
    left = number.clone()
    for j in range(3):
        part = torch.where(left > 0, torch.floor(left / torch.exp2(torch.floor(torch.log2(left.clamp_min(1))) - 3)) * torch.exp2(torch.floor(torch.log2(left.clamp_min(1))) - 3), 0.0).clamp(max=448)
        x[:, 1 + j] = x[:, 4 + j] = part
        left -= part
    assert (left == 0).all()                                                             # (up to 700: 448 and seven or eight bits more)
    ids = torch.randint(0, Ex, (M, 1), device="cuda", generator=gen(M), dtype=torch.int32)
    out = E.moe_fp8(ids, torch.ones(M, 1, device="cuda"), E.rec_table([rec] * Ex), 0, Ex, x.to(torch.bfloat16), H, I, out_dtype=torch.float32).double()
    s = (56.0 * 448.0 * 2.0 ** -9 * number / 448.0).float().double()[:, None]
    want = R.nearest_e4m3(torch.tensor([448.0] + mids, dtype=torch.float64, device="cuda")) * s
    n = len(mids) + 1
    assert torch.equal(out[:, :n], want.float().double()), ((out[:, :n] - want).abs() / want).max().item()
    assert (out[:, n:] == 0).all()


@pytest.mark.parametrize("N,dt", [((1 << 29) + 40, "float32"), (1 << 30, "bfloat16")])
def test_gemm_rows_of_the_result_beyond_31_bits_of_bytes(E, N, dt):
    """The most columns a product may have: what is left of a row is more than 2^31 bytes at its front."""
    import torch
    M, K, n = 33, 16, 700
    q = torch.zeros(N, K, dtype=torch.uint8, device="cuda")
    s = torch.ones(R.up(N), 1, device="cuda")
    part, ps = matrix(2 * n, K, 1)
    q[:n], q[-n:] = part[:n].view(torch.uint8), part[n:].view(torch.uint8)
    xq, xs = E.fp8_quant_rows(rows(M, K, M))
    y = torch.empty(M, N, dtype=getattr(torch, dt), device="cuda")
    y[:, :2 * n] = -7; y[:, -2 * n:] = -7
    E.fp8_gemm(E.GMat(E.FMT_FP8_B128, N, K, q, s), xq, xs, y=y)
    for cols, w in ((y[:, :n], part[:n]), (y[:, -n:], part[n:])):
        y0, a = R.gemm(R.codes_to_f64(xq), xs.double(), w.double(), torch.ones(R.up(n), 1, dtype=torch.float64, device="cuda"))
        tol = R.sum_bound(K) * a
        assert ((cols.double() - y0).abs() <= tol + R.HALF[y.dtype] * (y0.abs() + tol)).all()
    assert (y[:, n:2 * n] == 0).all() and (y[:, -2 * n:-n] == 0).all()
    del y, q
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", ["float32", "bfloat16"])
def test_moe_offsets_beyond_32_bits(E, dt):
    """Pairs' results more than 2^32 bytes from their first: the rows at the end are those of the formula."""
    import torch
    M, H, I, Ex, K = 70000, 8192, 128, 4, 4
    recs = [record(E, H, I, 10 * e) for e in range(Ex)]
    tab = E.rec_table([r[0] for r in recs])
    ids = torch.arange(M * K, device="cuda", dtype=torch.int32).view(M, K) % Ex
    w = torch.rand(M, K, device="cuda", generator=gen(1)) * 0.5
    x = torch.randn(M, H, device="cuda", generator=gen(2)).to(torch.bfloat16)
    assert M * K * H * 2 > 1 << 32
    out = E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, out_dtype=getattr(torch, dt))
    for at in (0, M - 40):
        sl = slice(at, at + 40)
        o0, tol, _ = R.moe(ids[sl], w[sl], [r[1] for r in recs], x[sl])
        tol = tol + (R.HALF[out.dtype] * (o0.abs() + tol) if dt == "bfloat16" else 0.0)
        assert ((out[sl].double() - o0).abs() <= tol + 1e-30).all()
    del out, x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M,Ex,K", [(400, 16, 4), (700, 100, 3), (300, 4, 2)])
def test_moe_long_lists_in_graphs_and_without_dependent_launches(E, M, Ex, K):
    """Lists of pairs that a kernel of their own puts in order, replayed with other inputs; and every kernel behind the one in front."""
    import torch
    H, I = 640, 256
    recs = [record(E, H, I, 10 * e)[0] for e in range(4)]
    tab = torch.tensor([recs[e % 4].data_ptr() for e in range(Ex)], dtype=torch.int64, device="cuda")
    ins = [(*routing(M, K, Ex, i), torch.randn(M, H, device="cuda", generator=gen(i)).to(torch.bfloat16)) for i in range(3)]
    call = lambda a, dt, ctx=None: E.moe_fp8(a[0], a[1], tab, 0, Ex, a[2], H, I, out_dtype=dt, ctx=ctx)
    for dt in (torch.float32, torch.bfloat16):
        ref = [call(a, dt) for a in ins]
        plain = E.Context(flags=E.HB_FLAG_NO_PDL)
        assert all(torch.equal(call(a, dt, plain), r) for a, r in zip(ins, ref))
        plain.check_device()
        buf = [t.clone() for t in ins[0]]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = call(buf, dt)
        for i in (1, 2, 0, 1):
            for b, t in zip(buf, ins[i]):
                b.copy_(t)
            g.replay()
            assert torch.equal(got, ref[i])
    E.context().check_device()


def test_moe_limit_and_gateless_shared(E):
    moe_check(E, 9, 512, 256, 6, 3, 1, limit=1.5, gate=False)
    moe_check(E, 200, 256, 128, 6, 3, 2, limit=0.7, shared=False)


@pytest.mark.parametrize("M,Ex,K", [(5, 6, 3), (60, 6, 3), (150, 4, 3)])
@pytest.mark.parametrize("limit", [0.0, 1.0])
def test_moe_rows_that_are_not_finite(E, M, Ex, K, limit):
    """NaN and infinities of a row come out as NaN in that row alone, clamped or not."""
    import torch
    H, I = 256, 256
    recs = [record(E, H, I, 10 * e) for e in range(Ex)]
    tab = E.rec_table([r[0] for r in recs])
    x = torch.randn(M, H, device="cuda", generator=gen(M)).to(torch.bfloat16)
    ids, w = routing(M, K, Ex, M)
    ref = E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, limit=limit, out_dtype=torch.float32)
    x[1, 200] = float("nan"); x[3, 0] = float("inf"); x[M - 1, 130] = -float("inf")
    out = E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, limit=limit, out_dtype=torch.float32)
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[[1, 3, M - 1]] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], ref[~bad])


def test_moe_hot_expert_missing_records_and_invalid_ids(E):
    import torch

    def edit(ids):
        ids[0, 1] = -1; ids[1, 0] = 7; ids[2, :] = -1; ids[3, :] = 1000                 # a row that nothing is left of, ids outside the table
    moe_check(E, 150, 256, 256, 7, 3, 3, hot=2, missing=(4,), edit=edit)
    moe_check(E, 12, 256, 256, 7, 3, 4, hot=2, missing=(4, 5), edit=edit)
    out = moe_check(E, 6, 256, 128, 5, 2, 5, missing=(0, 1, 2, 3, 4), shared=False)     # no record at all: nothing is added
    assert (out == 0).all()


def test_moe_the_same_expert_twice_in_a_row(E):
    def edit(ids):
        ids[:, 1] = ids[:, 0]
    moe_check(E, 30, 256, 128, 5, 3, 6, edit=edit)


def test_moe_rows_behind_the_last_and_layers(E):
    import torch
    H, I, Ex, K, M = 256, 256, 4, 2, 21
    recs = [record(E, H, I, 100 + e) for e in range(3 * Ex)]
    tab = E.rec_table([r[0] for r in recs])
    x = torch.randn(M, H, device="cuda", generator=gen(1)).to(torch.bfloat16)
    ids, w = routing(M, K, Ex, 2)
    for li in range(3):
        o0, tol, _ = R.moe(ids, w, [r[1] for r in recs[li * Ex:(li + 1) * Ex]], x)
        out = torch.full((M + 4, H), -7.0, device="cuda")
        E.moe_fp8(ids, w, tab, li, Ex, x, H, I, out=out[:M])
        assert ((out[:M].double() - o0).abs() <= tol).all() and (out[M:] == -7).all()


@pytest.mark.parametrize("M", [3, 40, 150])
def test_moe_misaligned_record_is_reported(E, M):
    """A record off its 16-byte boundary sets the device error word; the context works on."""
    import torch
    H, I, Ex, K = 256, 256, 4, 2
    buf = [torch.zeros(E.Fp8RecLayout(H, I).total + 64, dtype=torch.uint8, device="cuda") for _ in range(Ex)]
    recs = [record(E, H, I, 100 + e) for e in range(Ex)]
    x = torch.randn(M, H, device="cuda", generator=gen(1)).to(torch.bfloat16)
    ids, w = routing(M, K, Ex, 2)
    ids[0, 0] = 1
    ctx = E.Context()
    good = E.rec_table([r[0] for r in recs])
    ref = E.moe_fp8(ids, w, good, 0, Ex, x, H, I, ctx=ctx)
    ctx.check_device()
    for off in (1, 4, 8):
        bad = good.clone()
        bad[1] = buf[1].data_ptr() + 16 + off
        E.moe_fp8(ids, w, bad, 0, Ex, x, H, I, ctx=ctx)
        with pytest.raises(E.HbError, match="0x400000"):
            ctx.check_device()
        assert torch.equal(E.moe_fp8(ids, w, good, 0, Ex, x, H, I, ctx=ctx), ref)
        ctx.check_device()


def test_moe_refusals(E):
    import torch
    x = torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda")
    ids, w = routing(2, 2, 4, 1)
    tab = torch.zeros(4, dtype=torch.int64, device="cuda")
    for H, I in ((192, 256), (256, 192), (0, 128)):
        with pytest.raises(E.HbError):
            E.moe_fp8(ids, w, tab, 0, 4, x, H, I, out=torch.empty(2, 256, device="cuda"), ws=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))
    with pytest.raises(E.HbError):
        E.moe_fp8(ids, w, tab, 0, 1025, x, 256, 256)
    with pytest.raises(E.HbError):
        E.moe_fp8(ids, w, tab, -1, 4, x, 256, 256)
    with pytest.raises(E.HbError):
        E.moe_fp8(ids, w, tab, 0, 4, x, 256, 256, ws=torch.empty(1 << 22, dtype=torch.uint8, device="cuda")[16:])
    with pytest.raises(E.HbError):
        E.Fp8RecLayout(200, 128)
    assert E.moe_fp8(ids[:0], w[:0], tab, 0, 4, x[:0], 256, 256).shape == (0, 256)


def test_arguments_of_the_wrong_type_or_shape(E):
    import torch
    q, s = matrix(64, 256, 1)
    W = E.GMat(E.FMT_FP8_B128, 64, 256, q, s)
    xq, xs = E.fp8_quant_rows(rows(4, 256, 2))
    bf = dict(dtype=torch.bfloat16, device="cuda")
    calls = [lambda: E.fp8_gemm(W, xq, xs, y=torch.empty(4, 64, dtype=torch.float16, device="cuda")), lambda: E.fp8_gemm(W, xq, xs, y=torch.empty(3, 64, **bf)),
             lambda: E.fp8_gemm(W, xq, xs.double()), lambda: E.fp8_gemm(W, xq, xs[:1]), lambda: E.fp8_gemm(W, xq[:, :240], xs), lambda: E.fp8_gemm(W, xq.float(), xs),
             lambda: E.fp8_quant_rows(rows(4, 256, 2), q=torch.empty(3, 256, dtype=torch.uint8, device="cuda")), lambda: E.fp8_quant_rows(rows(4, 256, 2), s=torch.empty(2, 3, device="cuda")),
             lambda: E.fp8_quantize(rows(4, 256, 2), q=torch.empty(4, 512, dtype=torch.uint8, device="cuda")[:, ::2]),
             lambda: E.router_grouped_topk(torch.zeros(2, 64, **bf), 2), lambda: E.router_grouped_topk(torch.zeros(2, 64, device="cuda"), 2, bias=torch.zeros(63, device="cuda")),
             lambda: E.router_grouped_topk(torch.zeros(2, 64, device="cuda"), 2, ids=torch.zeros(1, 2, dtype=torch.int32, device="cuda")),
             lambda: E.router_grouped_topk(torch.zeros(2, 64, device="cuda"), 2, ids=torch.zeros(2, 2, dtype=torch.int64, device="cuda"))]
    x = torch.zeros(2, 256, **bf)
    ids, w = routing(2, 2, 4, 1)
    tab = torch.zeros(4, dtype=torch.int64, device="cuda")
    moe = lambda **k: E.moe_fp8(**{**dict(ids=ids, w=w, rec_tab=tab, li=0, E=4, x=x, H=256, I=256), **k})
    moe()
    calls += [lambda k=k: moe(**k) for k in (dict(ids=ids.long()), dict(w=w.double()), dict(w=w[:1]), dict(x=x.float()), dict(x=x[:, :128]), dict(x=x[:1]), dict(rec_tab=tab[:3]), dict(li=1),
                                             dict(out=torch.empty(1, 256, **bf)), dict(out=torch.empty(2, 256, dtype=torch.float16, device="cuda")), dict(shared=x[:1]), dict(shared=x.float()),
                                             dict(shared=x, lg=torch.zeros(2, 3, device="cuda"), col=3), dict(shared=x, lg=torch.zeros(2, 3, device="cuda"), col=-1), dict(shared=x, lg=x))]
    for c in calls:
        with pytest.raises(E.HbError):
            c()


# ---------------------------------------------------------------------------------------------------- together
def layer(E, lg, bias, x, tab, Ex, H, I, Wsh, K):
    """Router, routed experts, a dense matrix for every row beside them."""
    ids, w = E.router_grouped_topk(lg, K, 4, 2, bias=bias, scale=2.5)
    sh = E.fp8_gemm(Wsh, *E.fp8_quant_rows(x))
    return ids, w, E.moe_fp8(ids, w, tab, 0, Ex, x, H, I, shared=sh)


@pytest.mark.parametrize("M", [1, 11, 90])
def test_layer_on_streams_and_in_graphs(E, M):
    """Weights quantised here, routed, multiplied and summed; the same on another stream and replayed from a captured graph with other inputs."""
    import torch
    H, I, Ex, K = 512, 256, 16, 4
    g = gen(M)
    recs = [E.fp8_record(H, I, *(E.fp8_quantize(torch.randn(n, k, device="cuda", generator=g) * 0.05) for n, k in ((I, H), (I, H), (H, I)))) for _ in range(Ex)]
    tab = E.rec_table(recs)
    Wsh = E.GMat(E.FMT_FP8_B128, H, H, *E.fp8_quantize((torch.randn(H, H, device="cuda", generator=g) * 0.05).to(torch.bfloat16)))
    bias = torch.randn(Ex, device="cuda", generator=g) * 0.05
    ins = [(torch.randn(M, Ex, device="cuda", generator=g), torch.randn(M, H, device="cuda", generator=g).to(torch.bfloat16)) for _ in range(3)]
    ref = [layer(E, lg, bias, x, tab, Ex, H, I, Wsh, K) for lg, x in ins]
    L = E.Fp8RecLayout(H, I)
    parts = []
    for r in recs:
        parts.append([(r[a:a + n * k].view(torch.float8_e4m3fn).view(n, k).double(), r[b:b + n * k // 4096].view(torch.float32).view(n // 128, k // 128).double())
                      for a, b, n, k in ((L.w1, L.s1, I, H), (L.w3, L.s3, I, H), (L.w2, L.s2, H, I))])
    for (lg, x), (ids, w, out) in zip(ins, ref):
        i0, _ = R.route(lg.cpu().numpy(), bias.cpu().numpy(), K, 4, 2, 2, "sigmoid", True, 2.5)
        assert np.array_equal(ids.cpu().numpy(), i0)
        xq, xs = R.quant_rows(x.double())
        s0, a = R.gemm(xq, xs, Wsh.w.view(torch.float8_e4m3fn).double(), Wsh.s.double())
        o0, tol, _ = R.moe(ids, w, parts, x)
        tol = tol + R.sum_bound(H) * a + 2.0 ** -8 * s0.abs()
        o0 = o0 + s0
        assert ((out.double() - o0).abs() <= tol + 2.0 ** -8 * (o0.abs() + tol)).all()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for (lg, x), r in zip(ins, ref):
            got = layer(E, lg, bias, x, tab, Ex, H, I, Wsh, K)
            assert all(torch.equal(a, b) for a, b in zip(got, r))
    torch.cuda.current_stream().wait_stream(st)
    graphs = []
    for _ in range(2):                                                                   # two graphs, each with buffers of its own
        lg, x = ins[0][0].clone(), ins[0][1].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = layer(E, lg, bias, x, tab, Ex, H, I, Wsh, K)
        graphs.append((gr, lg, x, got))
    for i in (1, 2, 0):
        for gr, lg, x, got in graphs:
            lg.copy_(ins[i][0]); x.copy_(ins[i][1])
            gr.replay()
            assert all(torch.equal(a, b) for a, b in zip(got, ref[i]))
    E.context().check_device()

