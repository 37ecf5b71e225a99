"""GPU parity, routing limited to groups: ids equal to the 64-bit form's, weights within the fp32 bound, masks, ties and neighbours."""
import numpy as np
import pytest

import fp8_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    import eke_hive_b200 as E
    return E


def check(E, lg, bias, k, ng, tg, gt, score, renorm, scale):
    import torch
    ids, w = E.router_grouped_topk(torch.from_numpy(lg).cuda(), k, ng, tg, group_top=gt, score=score, bias=None if bias is None else torch.from_numpy(bias).cuda(),
                                   renorm=renorm, scale=scale)
    i0, w0 = R.route(lg, bias, k, ng, tg, gt, score, renorm, scale)
    i, w = ids.cpu().numpy(), w.cpu().numpy()
    bad = np.nonzero((i != i0).any(1))[0]
    assert bad.size == 0, (bad[:5], i[bad[:2]], i0[bad[:2]])
    tol = R.route_bound(lg, score) * np.abs(w0) + 2.0 ** -149
    assert (np.abs(w - w0) <= tol).all(), np.max(np.abs(w - w0) / (np.abs(w0) + 1e-30))
    return i, w


CASES = [(1, 256, 8, 8, 4, 2), (61, 160, 6, 8, 3, 1), (300, 256, 8, 8, 4, 2), (5, 1024, 16, 32, 5, 2), (7, 37, 3, 1, 1, 1), (9, 512, 10, 1, 1, 2), (33, 64, 8, 8, 1, 2), (4, 32, 1, 32, 7, 2),
         (3, 8, 8, 2, 2, 2), (2, 1, 1, 1, 1, 1), (130, 96, 5, 3, 2, 1), (17, 1024, 16, 2, 1, 2), (11, 24, 4, 8, 5, 2)]


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("M,Ex,k,ng,tg,gt", CASES)
def test_random(E, M, Ex, k, ng, tg, gt, score):
    rng = np.random.default_rng(M * 7 + Ex)
    for bias, renorm, scale in ((None, True, 1.0), (rng.normal(0, 0.1, Ex).astype(np.float32), True, 2.5), (rng.normal(0, 0.01, Ex).astype(np.float32), False, 16.0)):
        check(E, rng.normal(0, 1.5, (M, Ex)).astype(np.float32), bias, k, ng, tg, gt, score, renorm, scale)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_equal_scores_go_to_the_smaller_index(E, score):
    rng = np.random.default_rng(3)
    lg = (np.round(rng.normal(0, 1, (200, 256)) * 4) / 4).astype(np.float32)          # many equal logits
    check(E, lg, None, 8, 8, 4, 2, score, True, 2.5)
    check(E, lg, None, 8, 8, 4, 1, score, True, 2.5)
    check(E, lg, (np.round(rng.normal(0, 1, 256) * 2) / 64).astype(np.float32), 8, 8, 4, 2, score, True, 1.0)
    i, _ = check(E, np.zeros((3, 64), np.float32), None, 5, 4, 2, 2, score, True, 1.0)
    assert i.tolist() == [[0, 1, 2, 3, 4]] * 3


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("ng,tg", [(1, 1), (8, 3)])
def test_neighbours_that_fp32_scores_do_not_tell_apart(E, score, ng, tg):
    """Rows whose logits lie within a few fp32 steps of each other: the scores agree to fp32 precision, their order is the logits'."""
    rng = np.random.default_rng(5)
    base = rng.normal(0, 1, (64, 1)).astype(np.float32)
    lg = base.repeat(128, 1)
    step = np.spacing(np.abs(lg))
    lg = (lg + step * rng.permuted(np.tile(np.arange(128), (64, 1)), axis=1)).astype(np.float32)
    check(E, lg, None, 7, ng, tg, 2, score, True, 1.0)
    check(E, lg, None, 7, ng, tg, 1, score, False, 1.0)
    bias = (rng.integers(-3, 4, 128) * 2.0 ** -24).astype(np.float32)                 # and a bias of the same size as their distance
    check(E, lg, bias, 7, ng, tg, 2, score, True, 1.0)


@pytest.mark.parametrize("n", [2, 3, 9, 31, 32, 33, 60, 150])
@pytest.mark.parametrize("score,tied,better,best", [("sigmoid", 20.0, 25.0, 30.0), ("softmax", 1.0, np.nextafter(np.float32(1), np.float32(2)), 10.0), ("softmax", -np.inf, -100.0, 0.0),
                                                    ("sigmoid", -np.inf, -200.0, 0.0), ("sigmoid", -3e38, -120.0, 1.0)])
def test_a_better_expert_behind_a_tie_at_the_border(E, score, tied, better, best, n):
    """n equal logits, of which the picks take some, and behind them one that is better by less than fp32 scores show."""
    size = max(n + 2, 8)
    rng = np.random.default_rng(n)
    for Ex in (size, 256):
        lg = np.full((40, Ex), -np.inf if tied > -1e38 else tied, np.float32)
        for m in range(40):
            at = rng.permutation(Ex)[: n + 2]
            lg[m, at] = tied
            lg[m, max(at)] = better                                                   # (behind, by its index, all that it ties with in fp32)
            if m % 2:
                lg[m, at[0] if at[0] != max(at) else at[1]] = best
        for k in sorted({1, 2, min(n, 5), min(n, 16)}):
            check(E, lg, None, k, 1, 1, 1, score, False, 1.0)
    check(E, np.array([[20, 20, 25, 0]], np.float32), None, 1, 1, 1, 1, "sigmoid", False, 1.0)
    check(E, np.array([[1, 1, 1.0000001, 10]], np.float32), None, 2, 1, 1, 1, "softmax", False, 1.0)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("Ex,k,ng,tg,gt", [(256, 8, 8, 4, 2), (160, 6, 8, 3, 1), (64, 4, 1, 1, 1), (512, 10, 1, 1, 1), (1024, 16, 16, 9, 2), (24, 3, 1, 1, 1)])
def test_logits_as_a_bf16_product_leaves_them(E, score, Ex, k, ng, tg, gt):
    """Many equal logits, scores near the end of their range."""
    import torch
    rng = np.random.default_rng(Ex + k)
    for by in (1.0, 8.0, 30.0):
        lg = torch.from_numpy(np.clip(rng.normal(0, by, (700, Ex)), -30, 30).astype(np.float32)).to(torch.bfloat16).float().numpy()
        check(E, lg, None, k, ng, tg, gt, score, True, 2.5)
        check(E, lg, (rng.integers(-2, 3, Ex) * 2.0 ** -22).astype(np.float32), k, ng, tg, gt, score, False, 1.0)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_masks_and_extremes(E, score):
    rng = np.random.default_rng(6)
    lg = rng.normal(0, 1, (40, 64)).astype(np.float32)
    lg[0] = -np.inf                                                                   # nothing left
    lg[1] = np.nan
    lg[2, 1:] = -np.inf                                                               # one expert left
    lg[3, ::2] = -np.inf
    lg[4] = np.finfo(np.float32).min
    lg[5, 5:] = np.finfo(np.float32).min
    lg[6, 10] = np.nan
    lg[7] = 60.0 + rng.integers(0, 4, 64)                                             # sigmoid is 1 to 64 bits: ties
    lg[8] = -90.0 - rng.normal(0, 3, 64)                                              # scores far below fp32's normal range are still in order
    lg[9, 32:] = -np.inf
    lg[10:] *= 20
    bias = rng.normal(0, 0.2, 64).astype(np.float32)
    for b in (None, bias):
        for ng, tg in ((1, 1), (8, 2), (8, 8)):
            for gt in (1, 2):
                check(E, lg, b, 6, ng, tg, gt, score, False, 1.0)
                i, w = check(E, lg[9:], b, 6, ng, tg, gt, score, True, 1.0)
                assert all(len(set(r)) == 6 for r in i.tolist())


@pytest.mark.parametrize("Ex,k,ng,tg", [(64, 6, 8, 2), (64, 6, 1, 1), (20, 8, 10, 4), (1024, 16, 8, 4)])
def test_a_softmax_row_with_infinity_has_no_weights(E, Ex, k, ng, tg):
    """Its weights are NaN, as the header says, its picks are experts, all different; the rows beside it, and a sigmoid, take no harm."""
    import torch
    rng = np.random.default_rng(Ex)
    lg = rng.normal(0, 1, (9, Ex)).astype(np.float32)
    bad = lg.copy()
    bad[2, 3] = np.inf; bad[5, :] = np.inf; bad[7, -1] = np.inf; bad[7, 0] = np.nan
    ok = [0, 1, 3, 4, 6, 8]
    for bias in (None, rng.normal(0, 0.1, Ex).astype(np.float32)):
        b = None if bias is None else torch.from_numpy(bias).cuda()
        for renorm in (False, True):
            i0, w0 = R.route(lg, bias, k, ng, tg, 2, "softmax", renorm, 1.0)
            ids, w = E.router_grouped_topk(torch.from_numpy(bad).cuda(), k, ng, tg, score="softmax", bias=b, renorm=renorm)
            assert np.array_equal(ids.cpu().numpy()[ok], i0[ok]) and (np.abs(w.cpu().numpy()[ok] - w0[ok]) <= R.route_bound(lg, "softmax") * np.abs(w0[ok]) + 2.0 ** -149).all()
            assert torch.isnan(w[[2, 5, 7]]).all()
            assert all(len(set(r)) == k and min(r) >= 0 and max(r) < Ex for r in ids.tolist())
            check(E, bad, bias, k, ng, tg, 2, "sigmoid", renorm, 1.0)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("Ex,k,ng,tg", [(64, 6, 8, 2), (64, 6, 1, 1), (20, 8, 10, 4), (256, 8, 8, 4)])
def test_bias_that_is_not_finite(E, score, Ex, k, ng, tg):
    """Infinities count as the largest finite values and NaN as the lowest: picks are experts, all different, whatever the bias holds."""
    rng = np.random.default_rng(Ex)
    lg = rng.normal(0, 1, (30, Ex)).astype(np.float32)
    for n in (1, Ex // 2, Ex):
        bias = rng.normal(0, 0.1, Ex).astype(np.float32)
        bias[rng.permutation(Ex)[:n]] = rng.choice([np.nan, np.inf, -np.inf, np.finfo(np.float32).max], n)
        for gt in (1, 2):
            import torch
            ids, w = E.router_grouped_topk(torch.from_numpy(lg).cuda(), k, ng, tg, group_top=gt, score=score, bias=torch.from_numpy(bias).cuda())
            top = np.finfo(np.float32).max
            i0, w0 = R.route(lg, np.clip(np.where(np.isnan(bias), -top, bias), -top, top), k, ng, tg, gt, score, True, 1.0)
            assert np.array_equal(ids.cpu().numpy(), i0)
            assert (np.abs(w.cpu().numpy() - w0) <= R.route_bound(lg, score) * np.abs(w0) + 2.0 ** -149).all()


def test_row_stride_and_rows_behind_the_last(E):
    import torch
    rng = np.random.default_rng(8)
    lg = rng.normal(0, 1, (6, 70)).astype(np.float32)
    ids = torch.full((9, 4), -7, dtype=torch.int32, device="cuda")
    w = torch.full((9, 4), -7.0, device="cuda")
    E.router_grouped_topk(torch.from_numpy(lg).cuda(), 4, 4, 2, E=64, ids=ids, w=w)
    i0, w0 = R.route(lg[:, :64], None, 4, 4, 2, 2, "sigmoid", True, 1.0)
    assert np.array_equal(ids[:6].cpu().numpy(), i0) and np.abs(w[:6].cpu().numpy() - w0).max() <= 32 * 2.0 ** -24
    assert (ids[6:] == -7).all() and (w[6:] == -7).all()


def test_a_rows_result_does_not_depend_on_the_batch(E):
    import torch
    lg = torch.from_numpy(np.random.default_rng(9).normal(0, 1, (4000, 256)).astype(np.float32)).cuda()
    ids, w = E.router_grouped_topk(lg, 8, 8, 4, scale=2.5)
    for m0, n in ((0, 1), (17, 5), (100, 63), (1000, 700)):
        i1, w1 = E.router_grouped_topk(lg[m0:m0 + n], 8, 8, 4, scale=2.5)
        assert torch.equal(i1, ids[m0:m0 + n]) and torch.equal(w1, w[m0:m0 + n])


def test_refusals(E):
    import torch
    lg = torch.zeros(2, 64, device="cuda")
    for kw in (dict(k=0), dict(k=17), dict(k=9, n_group=8, topk_group=1), dict(k=2, n_group=0), dict(k=2, n_group=5), dict(k=2, n_group=33), dict(k=2, n_group=8, topk_group=9),
               dict(k=2, n_group=8, topk_group=0), dict(k=2, group_top=3), dict(k=2, group_top=0)):
        with pytest.raises(E.HbError):
            E.router_grouped_topk(lg, **kw)
    with pytest.raises(E.HbError):
        E.router_grouped_topk(torch.zeros(1, 1025, device="cuda"), 2)
    with pytest.raises(E.HbError):
        E.router_grouped_topk(lg, 2, E=65)
    ids, w = E.router_grouped_topk(lg[:0], 2)
    assert ids.shape == (0, 2)
