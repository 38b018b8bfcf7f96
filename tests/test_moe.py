"""The routed experts' MLP: refusals on the CPU, the GPU path against the
float64 oracle.  The tolerance is element-wise and derived (moe_mlp_bounds):
fp32 accumulation carried through the quantisation of h, and one rounding to
fp16."""
import ctypes

import numpy as np
import pytest
import torch


def _expert_weights(pkg, E, rows, K, g, scale_bytes=(2, 11)):
    codes = torch.randint(0, 256, (E, rows, K // 2), dtype=torch.uint8, generator=g)
    sf = torch.randint(*scale_bytes, (E, rows, K // 16), dtype=torch.uint8, generator=g)
    return codes, torch.stack([pkg.layout.to_blocked(s) for s in sf]), sf


class Problem:
    def __init__(self, pkg, T, k, E, D, F, seed=0, ids=None):
        g = torch.Generator().manual_seed(seed + T + 7 * E + D + F)
        self.x = torch.randn((T, D), generator=g).to(torch.float16)
        if ids is None:
            ids = torch.rand((T, max(E, k)), generator=g).argsort(dim=1)[:, :k] % E
        self.ids = ids.to(torch.int32).contiguous()
        self.weights = torch.softmax(torch.randn(self.ids.shape, generator=g), dim=1)
        self.wg, self.sg, self.sg_plain = _expert_weights(pkg, E, F, D, g)
        self.wu, self.su, self.su_plain = _expert_weights(pkg, E, F, D, g)
        self.wd, self.sd, self.sd_plain = _expert_weights(pkg, E, D, F, g)

    def args(self, dev="cuda"):
        return [t.to(dev) for t in (self.x, self.ids, self.weights, self.wg, self.wu, self.wd, self.sg, self.su, self.sd)]

    def check(self, oracle, got):
        want, tol = oracle.moe_mlp_bounds(self.x, self.ids, self.weights, self.wg, self.wu, self.wd, self.sg, self.su, self.sd)
        err = np.abs(got.cpu().double().numpy() - want)
        assert (err <= tol).all(), f"off by {err.max()} where {tol[np.unravel_index(err.argmax(), err.shape)]} is allowed"
        # the bound is worth something: most of it is the rounding to fp16
        if want.size:
            assert np.median(tol) < 0.05 * max(np.sqrt(np.mean(want ** 2)), 1e-3)


# ------------------------------------------------------------------- CPU

def test_oracle_moe_matches_its_quantiser(oracle):
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((20, 64)) * 2).astype(np.float16)
    codes, sf = oracle.quantize(x)
    np.testing.assert_array_equal(oracle.quantize_values(x), oracle.dequant_matrix(codes, sf, 20, 64).astype(np.float64))


def test_moe_refuses_without_gpu(pkg):
    l, p = pkg._lib.lib(), 4096
    need = ctypes.c_int64(0)
    ws = lambda *a: l.nvfp4_moe_workspace(*a, ctypes.byref(need))
    assert ws(4, 2, 8, 128, 128) == 0 and need.value > 0
    assert ws(0, 2, 8, 128, 128) == 0 and need.value == 0
    assert ws(-1, 2, 8, 128, 128) == 1 and ws(4, 0, 8, 128, 128) == 1 and ws(4, 33, 64, 128, 128) == 1
    assert ws(4, 2, 0, 128, 128) == 1 and ws(4, 2, 1025, 128, 128) == 1
    assert ws(4, 2, 8, 96, 128) == 1 and ws(4, 2, 8, 128, 0) == 1
    assert ws(1 << 24, 2, 8, 64, 64) == 1 and b"slots" in l.nvfp4_last_error()
    ws(4, 2, 8, 128, 128)

    def call(x=p, ldx=128, T=4, wg=p, ld=64, es=8192, sfe=1024, ldo=128, out=p, w=p, n=1 << 40):
        return l.nvfp4_moe_mlp(x, ldx, p, p, T, 2, 8, 128, 128, wg, p, p, p, ld, es, sfe, p, p, 64, 8192, 1024, out, ldo,
                               w, n, None)
    assert call(x=None) == 1 and call(w=None) == 1 and call(out=None) == 1 and call(wg=None) == 1
    assert call(x=p + 1) == 2 and call(out=p + 1) == 2 and call(w=p + 16) == 2 and call(wg=p + 8) == 2
    assert call(ldx=127) == 1 and call(ldo=100) == 1 and call(ld=48) == 1 and call(es=0) == 1 and call(sfe=-16) == 1
    assert call(ld=72) == 2 and call(es=8200) == 2
    assert call(n=need.value - 1) == 1 and b"workspace" in l.nvfp4_last_error()
    assert call(T=0, x=None) == 0


# ------------------------------------------------------------------- GPU

SHAPES = [
    (1, 2, 8, 512, 1024), (1, 1, 1, 64, 64), (5, 1, 3, 64, 64), (16, 8, 64, 256, 320), (64, 8, 16, 256, 192),
    (33, 3, 7, 192, 448), (100, 4, 8, 320, 576), (128, 1, 2, 128, 128), (129, 1, 1, 128, 128),
    (300, 2, 2, 256, 384), (333, 4, 8, 448, 320), (700, 2, 4, 192, 320), (3000, 2, 16, 64, 64), (40, 2, 300, 64, 128),
    (1000, 2, 2, 512, 768), (901, 1, 2, 256, 1024), (1500, 4, 5, 256, 256), (130, 6, 2, 768, 256),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,D,F", SHAPES)
def test_moe(pkg, oracle, cuda, T, k, E, D, F):
    p = Problem(pkg, T, k, E, D, F)
    out = pkg.moe_mlp(*p.args())
    torch.cuda.synchronize()
    assert pkg._lib.device_errors() == 0
    p.check(oracle, out)


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,D,F", [(60, 2, 32, 128, 192), (90, 4, 16, 128, 192), (500, 2, 4, 128, 192), (1000, 2, 4, 256, 256)])
def test_moe_everyone_wants_one_expert(pkg, oracle, cuda, T, k, E, D, F):
    g = torch.Generator().manual_seed(9)
    ids = torch.stack([torch.full((T,), E - 2)] + [torch.randint(0, E - 2, (T,), generator=g) for _ in range(k - 1)], dim=1)
    p = Problem(pkg, T, k, E, D, F, ids=ids)
    p.check(oracle, pkg.moe_mlp(*p.args()))
    assert pkg._lib.device_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,E", [(9, 8), (400, 4)])
def test_moe_skipped_and_repeated_slots(pkg, oracle, cuda, T, E):
    """Ids outside [0, E) are skipped, a token without any gets zeros, an
    expert twice in a row counts twice."""
    g = torch.Generator().manual_seed(8)
    ids = torch.randint(0, E, (T, 3), generator=g)
    ids[0] = -1
    ids[1, 1] = -1
    ids[2, 0] = E
    ids[3, 2] = 2 ** 31 - 1
    ids[4] = 1
    ids[T - 1] = -(2 ** 31)
    p = Problem(pkg, T, 3, E, 128, 128, ids=ids)
    out = pkg.moe_mlp(*p.args())
    p.check(oracle, out)
    assert (out[0] == 0).all() and (out[T - 1] == 0).all()


@pytest.mark.gpu
def test_moe_no_tokens_and_no_slots(pkg, oracle, cuda):
    p = Problem(pkg, 0, 2, 4, 64, 64)
    assert pkg.moe_mlp(*p.args()).shape == (0, 64)
    p = Problem(pkg, 6, 2, 4, 64, 64, ids=torch.full((6, 2), -1))
    assert (pkg.moe_mlp(*p.args()) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,E", [(12, 8), (600, 4)])
def test_moe_strides_and_dirty_memory(pkg, oracle, cuda, T, E):
    """Gate and up as halves of one merged tensor, padded expert strides, odd
    rows of x, an output with odd rows; memory that the allocator hands out
    holds NaN patterns; what lies around the output stays."""
    D, F, k = 192, 256, 2
    p = Problem(pkg, T, k, E, D, F)
    x, ids, w, wg, wu, wd, sg, su, sd = p.args()
    both = torch.cat([wg, wu], dim=1)
    sboth = torch.cat([sg, su], dim=1)
    pad = torch.full((E, D + 3, F // 2 + 16), 0xFF, dtype=torch.uint8, device=cuda)
    pad[:, :D, :F // 2] = wd
    bigx = torch.full((T, D + 7), float("nan"), dtype=torch.float16, device=cuda)
    bigx[:, 3:3 + D] = x
    bigo = torch.full((T + 2, D + 5), 3.0, dtype=torch.float16, device=cuda)
    need = ctypes.c_int64(0)
    pkg._lib.lib().nvfp4_moe_workspace(T, k, E, D, F, ctypes.byref(need))
    torch.cuda.synchronize()
    torch.full((need.value,), 0xFF, dtype=torch.uint8, device=cuda)     # freed at once: the next allocation is dirty
    out = pkg.moe_mlp(bigx[:, 3:3 + D], ids, w, both[:, :F], both[:, F:], pad[:, :D, :F // 2],
                      sboth[:, :sg.shape[1]], sboth[:, sg.shape[1]:], sd, out=bigo[1:T + 1, 1:1 + D])
    p.check(oracle, out)
    assert (bigo[[0, T + 1]] == 3).all() and (bigo[:, 0] == 3).all() and (bigo[:, D + 1:] == 3).all()
    assert pkg._lib.device_errors() == 0


@pytest.mark.gpu
def test_moe_plain_scales_types_and_in_place(pkg, oracle, cuda):
    p = Problem(pkg, 10, 2, 4, 128, 192)
    x, ids, w, wg, wu, wd = p.args()[:6]
    f8 = lambda s: s.to(cuda).view(torch.float8_e4m3fn)
    cast = (lambda t: t.view(torch.float4_e2m1fn_x2)) if hasattr(torch, "float4_e2m1fn_x2") else (lambda t: t)
    out = pkg.moe_mlp(x, ids, w, cast(wg), cast(wu), cast(wd), f8(p.sg_plain), f8(p.su_plain), f8(p.sd_plain), out=x)
    assert out.data_ptr() == x.data_ptr()
    p.check(oracle, out)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E", [(20, 8), (400, 2)])
def test_moe_graphs_and_streams(pkg, oracle, cuda, T, E):
    """Two captured graphs replayed on two streams at once, with new inputs in
    the captured buffers; the same calls bit for bit."""
    ps = [Problem(pkg, T, 2, E, 256, 256, seed=s) for s in (1, 2)]
    live = [p.args() for p in ps]
    want = [pkg.moe_mlp(*a).clone() for a in live]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in live:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pkg.moe_mlp(*a))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
    # other tokens and other experts through the same graph
    live[0][0].copy_(live[1][0])
    live[0][1].copy_((live[0][1] + 1) % E)
    graphs[0].replay()
    torch.cuda.synchronize()
    ps[0].x, ps[0].ids = ps[1].x, (ps[0].ids + 1) % E
    ps[0].check(oracle, outs[0])
    for p, w in zip(ps[1:], want[1:]):
        p.check(oracle, w)


@pytest.mark.gpu
def test_moe_calls_at_once(pkg, oracle, cuda):
    """Eager calls on three streams at once, of three sizes (each of the paths)."""
    ps = [Problem(pkg, 10, 2, 4, 256, 256, seed=3), Problem(pkg, 200, 2, 8, 256, 256, seed=4), Problem(pkg, 600, 2, 4, 256, 256, seed=5)]
    args = [p.args() for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    outs = [[], [], []]
    for _ in range(3):
        for o, s, a in zip(outs, streams, args):
            with torch.cuda.stream(s):
                o.append(pkg.moe_mlp(*a))
    torch.cuda.synchronize()
    for p, o in zip(ps, outs):
        p.check(oracle, o[0])
        assert all(torch.equal(o[0], x) for x in o[1:])
    assert pkg._lib.device_errors() == 0


@pytest.mark.gpu
def test_moe_rows_do_not_depend_on_the_batch_order(pkg, cuda):
    """The same tokens in another order, at the same sizes, give the same bits."""
    p = Problem(pkg, 300, 4, 8, 256, 256)
    a = p.args()
    perm = torch.randperm(300, generator=torch.Generator().manual_seed(1)).to(cuda)
    out = pkg.moe_mlp(*a)
    again = pkg.moe_mlp(a[0][perm], a[1][perm].contiguous(), a[2][perm].contiguous(), *a[3:])
    assert torch.equal(out[perm], again)


@pytest.mark.gpu
def test_moe_refusals(pkg, cuda):
    p = Problem(pkg, 4, 2, 4, 64, 128)
    a = p.args()

    def bad(i, t, err, match):
        b = list(a)
        b[i] = t
        with pytest.raises(err, match=match):
            pkg.moe_mlp(*b)
    bad(0, a[0].float(), TypeError, "float16")
    bad(0, a[0].cpu(), ValueError, "CUDA")
    bad(0, a[0][:, :32], ValueError, "expected")
    bad(1, a[1].long(), TypeError, "int32")
    bad(1, a[1][:3], ValueError, "ids")
    bad(2, a[2][:, :1], ValueError, "weights")
    bad(2, a[2].half(), TypeError, "float32")
    bad(4, a[4][:, :64], ValueError, "w_up")
    bad(5, a[3], ValueError, "w_down")
    bad(6, a[6][:, :10], ValueError, "scale_gate")
    bad(8, a[8].cpu(), ValueError, "device")
    with pytest.raises(ValueError, match="out"):
        pkg.moe_mlp(*a, out=torch.empty((4, 63), dtype=torch.float16, device=cuda))


@pytest.mark.gpu
def test_router_into_experts(pkg, oracle, cuda):
    """Router and experts together, as a layer uses them, with a masked expert
    and a token whose mask leaves one expert."""
    T, E, k, D, F = 50, 16, 4, 256, 320
    p = Problem(pkg, T, k, E, D, F)
    g = torch.Generator().manual_seed(12)
    wr = (torch.randn((E, D), generator=g) / D ** 0.5).to(cuda)
    a = p.args()
    logits = a[0].float() @ wr.t()
    logits[:, 5] = float("-inf")
    logits[7, 1:] = float("-inf")
    w, ids = pkg.route_experts(logits, k, score="sigmoid", bias=torch.randn(E, generator=g).to(cuda) * 0.1,
                               num_groups=4, top_groups=2, scale=1.5)
    out = pkg.moe_mlp(a[0], ids, w, *a[3:])
    torch.cuda.synchronize()
    p.ids, p.weights = ids.cpu(), w.cpu()
    assert (p.ids[7, 1:] == -1).all()
    p.check(oracle, out)


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E", [(5, 2, 4), (60, 4, 16), (300, 2, 2)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_moe_a_token_that_is_not_finite_stays_alone(pkg, cuda, T, k, E, bad):
    a = list(Problem(pkg, T, k, E, 192, 128).args())
    want = pkg.moe_mlp(*a)
    a[0] = a[0].clone()
    a[0][2] = bad
    got = pkg.moe_mlp(*a)
    keep = torch.arange(T, device=cuda) != 2
    assert torch.equal(got[keep], want[keep])
    assert pkg._lib.device_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 40])
def test_moe_most_experts_and_slots(pkg, oracle, cuda, T):
    p = Problem(pkg, T, 32, 1024, 64, 64)
    out = pkg.moe_mlp(*p.args())
    torch.cuda.synchronize()
    assert pkg._lib.device_errors() == 0
    p.check(oracle, out)


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,D,F", [
    (333, 4, 8, 192, 2048), (333, 4, 8, 192, 2112),      # both sides of the rule on the down product's tiles
    (384, 5, 8, 128, 128), (385, 5, 8, 128, 128), (384, 6, 8, 128, 128),   # and of that on the plan's launch
    (700, 2, 3, 1088, 64),
])
def test_moe_both_sides_of_the_rules(pkg, oracle, cuda, T, k, E, D, F):
    p = Problem(pkg, T, k, E, D, F)
    out = pkg.moe_mlp(*p.args())
    torch.cuda.synchronize()
    assert pkg._lib.device_errors() == 0
    p.check(oracle, out)


@pytest.mark.gpu
def test_moe_more_token_counts_than_maps_are_kept(pkg, oracle, cuda):
    """1100 token counts: four tensor maps of its workspace each, more than are kept at a time."""
    p = Problem(pkg, 1100, 1, 2, 64, 64)
    x, ids, w, *rest = p.args()
    want = pkg.moe_mlp(x, ids, w, *rest)
    p.check(oracle, want)
    for T in range(1, 1101):
        got = pkg.moe_mlp(x[:T], ids[:T], w[:T], *rest)
        if T % 50 == 0:
            assert torch.equal(got, pkg.moe_mlp(x[:T], ids[:T], w[:T], *rest))
    assert torch.equal(got, want)
    assert pkg._lib.device_errors() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,D,F", [
    (512, 4, 8, 128, 128), (512, 5, 8, 128, 128), (513, 1, 8, 128, 128), (513, 3, 8, 64, 128), (64, 32, 64, 64, 64),
    (1024, 1, 40, 64, 128),
])
def test_moe_both_sides_of_the_rule_on_the_plans_launch(pkg, oracle, cuda, T, k, E, D, F):
    p = Problem(pkg, T, k, E, D, F)
    out = pkg.moe_mlp(*p.args())
    torch.cuda.synchronize()
    assert pkg._lib.device_errors() == 0
    p.check(oracle, out)


def _digits(v, scales):
    """v = sum_b scales[b] * (sum of 15 e2m1 values): the codes [len(scales), 15], coarsest scale first."""
    grid = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    out = np.zeros((len(scales), 15), np.int64)
    for b, s in enumerate(scales):
        m = np.clip(np.round(v / s * 2) / 2, -84, 84)        # a multiple of 0.5
        v -= m * s
        left = abs(m)
        for j in range(15):
            c = int(np.searchsorted(grid, left, side="right")) - 1
            out[b, j] = c | (8 if m < 0 and c else 0)
            left -= grid[c]
        assert left == 0
    assert v == 0
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [1, 40])
def test_moe_values_beside_the_borders_of_codes(pkg, cuda, copies):
    """Gate and up products that are exact in 32 bits and whose silu(g) * u lies between 12.4 and 13.8 units of 2^-24 from
    the border of two codes, a little more than the error that SiLU in 32 bits may have: h must get the code of the exact
    value.  The down product is the identity, so the output is h as quantised.  Both forms (16 tokens, 640 tokens of 16
    experts)."""
    E, D = 16, 128
    unit, scale = 2.0 ** -24, 2.0 ** -9                       # of h's blocks
    scales = [2.0 ** 8, 2.0 ** 1, 2.0 ** -6, 2.0 ** -9]
    silu = lambda g: g / (1 + np.exp(-g))
    # g where g * log2(e) rounds far down, so that an exponential of the rounded product is off the most
    g = -np.arange(17 * 1024, 20 * 1024) / 1024.0
    t = (g.astype(np.float32) * np.float32(-1.4426950408889634)).astype(np.float64)
    g = g[np.argsort((t - g * -1.4426950408889634))][:E * 120]
    pairs, want = np.zeros((E, D, 2)), np.zeros((E, D))
    borders, values = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5]), np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    at = beside = 0
    for e in range(E):
        for c in range(D):
            if c % 16 == 0:                                   # its amax fixes the block's scale
                pairs[e, c] = -12.0, np.round(6 * scale / silu(-12.0) * 1024) / 1024
            else:
                reach = borders[(borders * scale / -silu(g[at]) < 21000)]
                u = reach[-1] * scale / silu(g[at])           # negative: h is positive
                near = (np.floor(u * (1 - 13.1 * unit) * 1024) + np.arange(-9, 10)) / 1024
                off = 1 - near / u
                fit = near[(off > 12.4 * unit) & (off < 13.8 * unit)]
                beside += len(fit) > 0
                pairs[e, c] = g[at], fit[0] if len(fit) else np.round(u * 0.97 * 1024) / 1024   # u's grid is too coarse there
                at += 1
            v = silu(pairs[e, c, 0]) * pairs[e, c, 1] / scale
            want[e, c] = values[np.searchsorted(borders, v)] * scale
    assert beside > 1000
    codes = np.zeros((2, E, D, D), np.int64)
    for m in range(2):
        for e in range(E):
            for c in range(D):
                d = _digits(pairs[e, c, m], scales)
                for b in range(4):
                    codes[m, e, c, 16 * b + 1:16 * b + 16] = d[b]
    pack = lambda c: torch.from_numpy((c[..., 0::2] | c[..., 1::2] << 4).astype(np.uint8)).to(cuda)
    e4m3 = lambda v: torch.tensor(v, dtype=torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
    sf = e4m3(scales + [1.0] * 4).repeat(E, D, 1).to(cuda)
    eye = torch.zeros((E, D, D), dtype=torch.int64)
    eye[:, torch.arange(D), torch.arange(D)] = 2              # 1.0
    x = torch.ones((E * copies, D), dtype=torch.float16, device=cuda)
    x[:, ::16] = 6.0                                          # a scale of 1; the weights there are 0
    ids = torch.arange(E, dtype=torch.int32, device=cuda).repeat(copies).unsqueeze(1).contiguous()
    one = torch.full((E, D, D // 16), 0x38, dtype=torch.uint8, device=cuda)
    out = pkg.moe_mlp(x, ids, torch.ones((E * copies, 1), device=cuda), pack(codes[0]), pack(codes[1]), pack(eye.numpy()),
                      sf, sf, one)
    got = out.cpu().double().numpy().reshape(copies, E, D)
    assert (got == want).all(), f"{(got != want).sum()} of {got.size} codes"
