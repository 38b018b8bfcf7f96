"""Routing of tokens to experts: refusals on the CPU, and the GPU kernel against
the float64 oracle (ids equal, weights within 32-bit rounding).

Weights tolerance: with logits within 32 of the row's maximum an exponential is
off by at most (32 + 2) * 2^-24 (argument rounding and the function itself), a
sum of up to 1024 terms adds at most 37 roundings, the quotients and the scale
four more on each side: (34 + 37 + 8) * 2^-24 < 6e-6."""
import math

import numpy as np
import pytest
import torch

RTOL, ATOL = 6e-6, 1e-37


def _check(pkg, oracle, logits, k, bias=None, **kw):
    w, ids = pkg.route_experts(logits, k, bias=bias, **{"num_groups": kw.get("groups", 1), **{a: b for a, b in kw.items() if a != "groups"}})
    torch.cuda.synchronize()
    rw, ri = oracle.route(logits, k, bias, **kw)
    np.testing.assert_array_equal(ids.cpu().numpy(), ri)
    np.testing.assert_allclose(w.cpu().numpy().astype(np.float64), rw, rtol=RTOL, atol=ATOL)
    return w, ids


# ------------------------------------------------------------------- CPU

def test_oracle_route_by_hand(oracle):
    x = np.array([[0.0, math.log(3.0), -np.inf, math.log(2.0)]])
    w, ids = oracle.route(x, 2)
    assert ids.tolist() == [[1, 3]]
    np.testing.assert_allclose(w, [[0.6, 0.4]])
    w, ids = oracle.route(x, 4, renormalize=False, scale=2.0)
    assert ids.tolist() == [[1, 3, 0, -1]]
    np.testing.assert_allclose(w, [[1.0, 2 / 3, 1 / 3, 0.0]])
    # groups {0,1} and {2,3}: sums 1/2 + 3/4 against 2/3 + nothing
    w, ids = oracle.route(x, 2, score="sigmoid", groups=2, top_groups=1)
    assert ids.tolist() == [[1, 0]]
    np.testing.assert_allclose(w, [[0.6, 0.4]])


def test_route_refuses_without_gpu(pkg):
    l, p = pkg._lib.lib(), 4096
    call = lambda T=4, E=8, ld=8, score=0, k=2, g=1, tg=1, gt=2, dt=0, x=p, w=p: l.nvfp4_route_experts(
        x, dt, T, E, ld, None, score, k, g, tg, gt, 1, 1.0, w, p, None)
    assert call(E=0) == 1 and call(E=1025, ld=1025) == 1
    assert call(k=0) == 1 and call(k=9) == 1 and call(E=64, ld=64, k=33) == 1
    assert call(g=3) == 1 and call(tg=2) == 1 and call(tg=0) == 1 and call(E=64, ld=64, g=64) == 1
    assert call(gt=3) == 1 and call(gt=0) == 1 and call(score=2) == 1 and call(dt=3) == 1 and call(ld=7) == 1
    assert call(x=None) == 1 and b"null" in l.nvfp4_last_error()
    assert call(x=p + 2) == 2 and call(w=p + 2) == 2
    assert call(T=0, x=None) == 0
    with pytest.raises(ValueError, match="CUDA"):
        pkg.route_experts(torch.zeros(2, 8), 2)
    with pytest.raises(TypeError):
        pkg.route_experts(torch.zeros(2, 8, dtype=torch.float64), 2)


# ------------------------------------------------------------------- GPU

CASES = [
    (1, 8, 2, {}), (3, 1, 1, {}), (5, 2, 2, {}), (257, 7, 3, {}), (33, 32, 32, {}), (64, 60, 4, {}),
    (40, 128, 8, dict(renormalize=False, scale=1.7)), (20, 1000, 8, {}), (9, 1024, 32, dict(renormalize=False)),
    (64, 256, 8, dict(groups=8, top_groups=4)), (31, 256, 8, dict(groups=8, top_groups=4, group_top=1)),
    (50, 60, 4, dict(groups=4, top_groups=2)), (50, 96, 6, dict(groups=32, top_groups=5)),
    (50, 64, 8, dict(groups=32, top_groups=4)), (17, 512, 9, dict(groups=2, top_groups=2)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,kw", CASES)
def test_route(pkg, oracle, cuda, T, E, k, kw, dtype, with_bias, score):
    g = torch.Generator().manual_seed(T * 1000 + E)
    x = (torch.randn((T, E), generator=g) * 2).to(dtype).to(cuda)
    bias = (torch.randn(E, generator=g) * 0.1).to(cuda) if with_bias else None
    _check(pkg, oracle, x, k, bias, score=score, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_masked_and_special_values(pkg, oracle, cuda, groups, with_bias, score):
    """Rows whose mask leaves nothing or fewer than k, NaN, infinities, the
    type's lowest value, signed zeros, rows of equal logits."""
    E, k = 16, 5
    g = torch.Generator().manual_seed(3)
    x = torch.randn((12, E), generator=g)
    low = torch.finfo(torch.float32).min
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = low
    x[3, 3:] = -math.inf
    x[4, ::2] = math.nan
    x[5, 7] = math.inf
    x[5, 2] = math.inf
    x[6] = 0.0
    x[6, 1::2] = -0.0
    x[7] = 1.25
    x[8, 4:] = low
    x[9, :8] = -math.inf
    x[10, :13] = -math.inf
    x[11] = x[11] * 30
    bias = None
    if with_bias:
        bias = torch.randn(E, generator=g) * 0.1
        bias[1], bias[6], bias[9], bias[12] = -math.inf, math.nan, 0.5, 0.5
        bias = bias.to(cuda)
    _check(pkg, oracle, x.to(cuda), k, bias, score=score, groups=groups, top_groups=max(1, groups // 2))


@pytest.mark.gpu
def test_route_infinite_bias_ranks_first(pkg, oracle, cuda):
    x = torch.randn((6, 8), generator=torch.Generator().manual_seed(4)).to(cuda)
    bias = torch.zeros(8)
    bias[3] = bias[5] = math.inf
    w, ids = _check(pkg, oracle, x, 3, bias.to(cuda), score="sigmoid")
    assert (ids[:, 0] == 3).all() and (ids[:, 1] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("gap", [0.0, 1e-8, 1e-6, 1e-5])
def test_route_near_ties_are_ranked_in_64_bits(pkg, oracle, cuda, gap, score):
    """Choices that differ by less than 32-bit arithmetic can tell: the bias
    makes every expert's choice the same up to `gap` and the bias's rounding."""
    E, T = 64, 50
    g = torch.Generator().manual_seed(5)
    x = torch.randn(E, generator=g)
    s = torch.softmax(x.double(), 0) if score == "softmax" else torch.sigmoid(x.double())
    bias = (0.75 - s + gap * torch.rand(E, generator=g)).float()
    _check(pkg, oracle, x.repeat(T, 1).to(cuda), 8, bias.to(cuda), score=score, groups=4, top_groups=2)
    _check(pkg, oracle, x.repeat(T, 1).to(cuda), 8, bias.to(cuda), score=score)


@pytest.mark.gpu
def test_route_strided_rows_other_stream_and_outputs(pkg, oracle, cuda):
    g = torch.Generator().manual_seed(6)
    big = torch.randn((40, 77), generator=g).to(cuda)
    x = big[:, 3:67]
    w = torch.full((42, 4), 7.0, device=cuda)
    ids = torch.full((42, 4), 7, dtype=torch.int32, device=cuda)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        pkg.route_experts(x, 4, weights=w[1:41], ids=ids[1:41])
    torch.cuda.synchronize()
    rw, ri = oracle.route(x, 4)
    np.testing.assert_array_equal(ids[1:41].cpu().numpy(), ri)
    np.testing.assert_allclose(w[1:41].cpu().numpy(), rw, rtol=RTOL, atol=ATOL)
    assert (w[[0, 41]] == 7).all() and (ids[[0, 41]] == 7).all()     # rows around stay as they were


@pytest.mark.gpu
def test_route_no_tokens_and_many(pkg, oracle, cuda):
    w, ids = pkg.route_experts(torch.empty((0, 8), device=cuda), 2)
    assert w.shape == (0, 2) and ids.shape == (0, 2)
    x = torch.randn((20000, 16), generator=torch.Generator().manual_seed(7)).to(cuda)
    _check(pkg, oracle, x, 2)


@pytest.mark.gpu
def test_route_refusals(pkg, cuda):
    x = torch.zeros((4, 8), device=cuda)
    with pytest.raises(RuntimeError, match="top_k"):
        pkg.route_experts(x, 9)
    with pytest.raises(RuntimeError, match="groups"):
        pkg.route_experts(x, 2, num_groups=3)
    with pytest.raises(ValueError, match="score"):
        pkg.route_experts(x, 2, score="relu")
    with pytest.raises(ValueError, match="bias"):
        pkg.route_experts(x, 2, bias=torch.zeros(7, device=cuda))
    with pytest.raises(ValueError, match="contiguous"):
        pkg.route_experts(torch.zeros((8, 4), device=cuda).t(), 2)
    with pytest.raises(ValueError, match="ids"):
        pkg.route_experts(x, 2, ids=torch.zeros((4, 2), dtype=torch.int64, device=cuda))


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("T,E,k,groups,top_groups,off", [
    (20001, 256, 8, 8, 4, 0), (10007, 256, 3, 16, 2, 0), (9600, 128, 8, 1, 1, 1), (40001, 32, 2, 32, 5, 0), (9500, 64, 16, 4, 3, 4),
    (9777, 60, 4, 1, 1, 0), (9600, 160, 6, 20, 3, 0)])
def test_route_many_rows(pkg, oracle, cuda, T, E, k, groups, top_groups, off, with_bias, dtype, score):
    """Enough rows for a warp to take several at once; some masked, equal or
    far apart among them, and an unaligned row start."""
    g = torch.Generator().manual_seed(T + E)
    x = torch.randn((T, E + off), generator=g).mul(2).to(dtype)
    x[5::97, ::3] = -math.inf
    x[6::97] = 0.5
    x[7::97, 1::2] = -1000.0
    x[8::97, 4:9] = 3.0
    x[9::97] = math.nan
    bias = (torch.randn(E, generator=g) * 0.1).to(cuda) if with_bias else None
    x = x.to(cuda)[:, off:]
    w, ids = pkg.route_experts(x, k, bias=bias, score=score, num_groups=groups, top_groups=top_groups)
    rows = torch.unique(torch.cat([torch.arange(0, T, 61), torch.arange(5, T, 97), torch.arange(6, T, 97),
                                   torch.arange(7, T, 97), torch.arange(8, T, 97), torch.arange(9, T, 97), torch.tensor([T - 1])]))
    rw, ri = oracle.route(x[rows.to(cuda)], k, bias, score=score, groups=groups, top_groups=top_groups)
    np.testing.assert_array_equal(ids[rows.to(cuda)].cpu().numpy(), ri)
    np.testing.assert_allclose(w[rows.to(cuda)].cpu().numpy().astype(np.float64), rw, rtol=RTOL, atol=ATOL)


@pytest.mark.gpu
def test_route_refuses_outputs_that_are_no_tensors(pkg, cuda):
    x = torch.zeros((4, 8), device=cuda)
    with pytest.raises(ValueError, match="weights"):
        pkg.route_experts(x, 2, weights=[0.0] * 8)
    with pytest.raises(ValueError, match="ids"):
        pkg.route_experts(x, 2, ids=[0] * 8)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["plain", "bias", "groups", "unscaled"])
@pytest.mark.parametrize("E,k", [(96, 5), (128, 8), (256, 8), (250, 32), (500, 12), (1024, 9)])
def test_route_equal_logits_of_one_lane(pkg, oracle, cuda, E, k, kind, dtype, score):
    """Equal logits 32 experts apart, which one lane of a warp ranks, with larger ones behind, between and before them:
    ties go to the lowest index."""
    g = torch.Generator().manual_seed(E + k)
    T = 60
    x = torch.randint(0, 5, (T, E), generator=g).float() / 2     # many ties everywhere
    x[0] = -4
    x[0, [3, 35]], x[0, 67] = 1.0, 2.0                           # two equal ones, then a larger one
    x[1] = torch.randn(E, generator=g) - 4
    x[1, 1::32] = 1.0
    x[1, E - 31:E:32] = 2.0
    x[2:20] = torch.randn((18, E), generator=g) - 4              # ties in a few lanes alone
    for t in range(2, 20):
        lane = int(torch.randint(0, 32, (1,), generator=g))
        x[t, lane::32] = torch.randint(1, 4, (len(x[t, lane::32]),), generator=g).float()
    kw = dict(score=score)
    bias = torch.zeros(E, device=cuda) if kind == "bias" else None
    if kind == "groups":
        kw.update(groups=2, top_groups=1) if E % 2 == 0 else None
    if kind == "unscaled":
        kw.update(renormalize=False)
    _check(pkg, oracle, x.to(dtype).to(cuda), k, bias, **kw)


@pytest.mark.gpu
def test_route_ties_in_many_rows(pkg, oracle, cuda):
    """bfloat16 logits of a long prompt, of few different values: every row's ids."""
    x = (torch.randn((12000, 256), generator=torch.Generator().manual_seed(11)) * 2).to(torch.bfloat16)
    x[::2] = (x[::2].float() * 2).round().div(2).to(torch.bfloat16)
    _, ids = pkg.route_experts(x.to(cuda), 8)
    want = x.float().sort(dim=1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(ids.cpu().long(), want)


# Scores that 32 bits cannot hold although the weights made of them are ordinary numbers.  Tolerance: an exponential of
# an argument up to 88 away is off by at most (88 + 2) * 2^-24 where 32 bits still do, the sum and the quotients as above:
# (90 + 37 + 8) * 2^-24 < 8.1e-6.  A weight of less than 64 times the smallest normal number (7.6e-37) may be lost.
FAINT_RTOL, FAINT_ATOL = 8.1e-6, 7.6e-37


def _check_weights(oracle, got, logits, k, bias=None, rows=None, **kw):
    w, ids = (t.cpu() for t in got)
    rows = torch.arange(len(logits)) if rows is None else rows
    rw, ri = oracle.route(logits.cpu()[rows], k, bias, **kw)
    np.testing.assert_array_equal(ids[rows].numpy(), ri)
    np.testing.assert_allclose(w[rows].numpy().astype(np.float64), rw, rtol=FAINT_RTOL, atol=FAINT_ATOL)
    return rw


@pytest.mark.gpu
@pytest.mark.parametrize("E,k,groups,top_groups", [(8, 2, 1, 1), (60, 5, 1, 1), (256, 8, 1, 1), (256, 8, 8, 4), (96, 3, 4, 1), (400, 4, 1, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("T", [41, 9700])
def test_route_sigmoids_below_32_bits(pkg, oracle, cuda, T, with_bias, dtype, E, k, groups, top_groups):
    """Rows of logits around -80 to -700: every score is tiny, their ratios are not.  Few rows and enough for a warp to
    take several at once."""
    g = torch.Generator().manual_seed(T + E)
    x = (torch.randn((T, E), generator=g) * 3 - torch.linspace(80, 690, T)[torch.randperm(T, generator=g)].unsqueeze(1)).to(dtype)
    x[::7] += 690                                                # ordinary rows among them
    x[3::7, 1:] -= 5                                             # one expert far above the others
    bias = torch.randn(E, generator=g).to(cuda) if with_bias else None
    got = pkg.route_experts(x.to(cuda), k, bias=bias, score="sigmoid", num_groups=groups, top_groups=top_groups, scale=2.5)
    rows = torch.arange(0, T, 1 if T < 100 else 23)
    rw = _check_weights(oracle, got, x, k, bias, rows, score="sigmoid", groups=groups, top_groups=top_groups, scale=2.5)
    np.testing.assert_allclose(rw.sum(axis=1), 2.5)              # no row was lost in 64 bits


@pytest.mark.gpu
@pytest.mark.parametrize("E,k,groups,top_groups", [(8, 2, 1, 1), (60, 5, 1, 1), (256, 8, 1, 1), (256, 8, 8, 4), (96, 3, 4, 1), (400, 4, 1, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [41, 9700])
def test_route_bias_prefers_experts_far_below(pkg, oracle, cuda, T, dtype, E, k, groups, top_groups):
    """A softmax whose bias keeps the larger half of the logits out: the chosen scores are e^-80 to e^-600 of the
    largest."""
    g = torch.Generator().manual_seed(T + E + 1)
    x = torch.randn((T, E), generator=g)
    x[:, :E // 2] += torch.linspace(80, 600, T)[torch.randperm(T, generator=g)].unsqueeze(1)
    x[::7, :E // 2] = 0
    x = x.to(dtype)
    bias = torch.randn(E, generator=g)
    bias[:E // 2] -= 20
    got = pkg.route_experts(x.to(cuda), k, bias=bias.to(cuda), num_groups=groups, top_groups=top_groups)
    rows = torch.arange(0, T, 1 if T < 100 else 23)
    rw = _check_weights(oracle, got, x, k, bias, rows, groups=groups, top_groups=top_groups)
    np.testing.assert_allclose(rw.sum(axis=1), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("scale", [1.0, 1e30])
def test_route_weights_that_a_scale_brings_back(pkg, oracle, cuda, scale, renormalize, with_bias):
    x = torch.randn((50, 24), generator=torch.Generator().manual_seed(3)) - torch.linspace(0, 160, 50).unsqueeze(1)
    bias = torch.randn(24, generator=torch.Generator().manual_seed(4)).to(cuda) if with_bias else None
    got = pkg.route_experts(x.to(cuda), 6, bias=bias, score="sigmoid", renormalize=renormalize, scale=scale)
    _check_weights(oracle, got, x, 6, bias, score="sigmoid", renormalize=renormalize, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k,groups,top_groups", [
    (9471, 64, 4, 1, 1), (9472, 64, 4, 1, 1), (9473, 200, 5, 1, 1), (12000, 200, 4, 1, 1), (9600, 256, 8, 8, 4), (9600, 256, 9, 8, 4)])
def test_route_both_sides_of_the_rule_on_ties(pkg, oracle, cuda, T, E, k, groups, top_groups, dtype, score):
    x = (torch.randn((T, E), generator=torch.Generator().manual_seed(T + k)) * 2).to(dtype)
    x[::2] = (x[::2].float() * 4).round().div(4).to(dtype)       # half of the rows with many ties
    w, ids = pkg.route_experts(x.to(cuda), k, score=score, num_groups=groups, top_groups=top_groups)
    rows = torch.cat([torch.arange(0, T, 31), torch.tensor([T - 1])])
    rw, ri = oracle.route(x[rows], k, score=score, groups=groups, top_groups=top_groups)
    np.testing.assert_array_equal(ids.cpu()[rows].numpy(), ri)
    np.testing.assert_allclose(w.cpu()[rows].numpy().astype(np.float64), rw, rtol=RTOL, atol=ATOL)
