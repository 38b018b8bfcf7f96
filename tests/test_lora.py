"""Low-rank adapters: refusals on the CPU, the GPU kernels against the float64
oracle with its derived element-wise tolerance (fp32 sums, one rounding)."""
import ctypes

import numpy as np
import pytest
import torch


class Problem:
    def __init__(self, T, K, N, r, n, run=1, mixed=True, seed=0):
        g = torch.Generator().manual_seed(seed + T + K + N + r)
        h = lambda *s: torch.randn(s, generator=g).to(torch.float16)
        self.x, self.base = h(T, K), h(T, N)
        self.a = (h(n, r, K).float() / K ** 0.5).to(torch.float16)
        self.b = (h(n, N, r).float() / r ** 0.5).to(torch.float16)
        owner = torch.randint(-1, n, (-(-max(T, 1) // run),), generator=g)
        self.adapters = owner.repeat_interleave(run)[:T].to(torch.int32).contiguous()
        self.scales = torch.rand(n, generator=g) + 0.5 if mixed else None
        self.ranks = torch.randint(0, r + 1, (n,), generator=g).to(torch.int32) if mixed else None
        if mixed:
            self.ranks[0] = r
            for i in range(n):      # what lies beyond a rank may hold anything
                self.a[i, self.ranks[i]:] = float("nan")
                self.b[i, :, self.ranks[i]:] = float("inf")

    def args(self, dev="cuda"):
        mv = lambda t: None if t is None else t.to(dev)
        return [mv(t) for t in (self.base, self.x, self.a, self.b, self.adapters, self.scales, self.ranks)]

    def check(self, oracle, got):
        want, tol = oracle.lora_add(self.base, self.x, self.a, self.b, self.adapters, self.scales, self.ranks)
        err = np.abs(got.cpu().double().numpy() - want)
        assert (err <= tol).all(), f"off by {err.max()}, {(~(err <= tol)).sum()} elements"


# ------------------------------------------------------------------- CPU

def test_oracle_lora_by_hand(oracle):
    t = lambda *v: torch.tensor(v, dtype=torch.float64)
    a = t(1, 2, 3, 4).view(1, 2, 2)
    b = t(1, 0, 0, 1, 1, 1).view(1, 3, 2)
    out, _ = oracle.lora_add(t(1, 1, 1).view(1, 3), t(1, -1).view(1, 2), a, b, torch.tensor([0]), t(2))
    assert out.tolist() == [[1 - 2, 1 - 2, 1 - 4]]
    out, _ = oracle.lora_add(t(1, 1, 1).view(1, 3), t(1, -1).view(1, 2), a, b, torch.tensor([0]), None, torch.tensor([1]))
    assert out.tolist() == [[0, 1, 0]]


def test_lora_refuses_without_gpu(pkg):
    l, p = pkg._lib.lib(), 4096
    need = ctypes.c_int64(-1)
    ws = lambda *a: l.nvfp4_lora_workspace(*a, ctypes.byref(need))
    assert ws(1, 16, 4) == 0 and need.value == 0
    assert ws(5000, 64, 4) == 0 and need.value > 0
    assert ws(-1, 16, 4) == 1 and ws(4, 8, 4) == 1 and ws(4, 24, 4) == 1 and ws(4, 144, 4) == 1
    assert ws(4, 16, 0) == 1 and ws(4, 16, 1024) == 1 and b"adapters" in l.nvfp4_last_error()

    far = p + (1 << 30)

    def call(base=p, ldb=16, x=far, ldx=64, lda=64, sa=1024, T=4, K=64, r=16, n=2, out=p, ldo=100, N=100, ldbase=100,
             w=None, wb=0, ad=p):
        return l.nvfp4_lora_add(base, ldbase, x, ldx, p, lda, sa, p, ldb, 1600, ad, None, None, T, K, N, r, n, out, ldo,
                                w, wb, None)
    assert call(base=None) == 1 and call(x=None) == 1 and call(out=None) == 1
    assert call(K=60) == 1 and call(N=0) == 1 and call(K=0) == 1
    assert call(ldx=56) == 1 and call(ldo=99, out=p + 2) == 1 and call(ldbase=99, out=p + 2) == 1 and call(lda=32) == 1
    assert call(sa=-8) == 1 and call(ldb=8) == 1
    assert call(x=far + 8) == 2 and call(ldx=68) == 2 and call(sa=1028) == 2 and call(base=p + 1, out=p) == 2
    assert call(ad=p + 2) == 2
    assert call(ldo=104) == 1 and b"stride" in l.nvfp4_last_error()          # in place with another row stride
    assert call(T=5000) == 1 and b"workspace" in l.nvfp4_last_error()
    assert call(T=5000, w=p, wb=64) == 1
    assert call(T=0, base=None) == 0
    # out over x, out over a shifted base; column slices of one buffer do not meet
    assert call(x=p, ldx=104, ldbase=104, ldo=104) == 1 and b"overlaps x" in l.nvfp4_last_error()
    assert call(x=p + 96, ldx=152, ldbase=152, ldo=152) == 1 and b"overlaps x" in l.nvfp4_last_error()
    assert call(out=p + 2, ldo=104, ldbase=104) == 1 and b"overlaps base" in l.nvfp4_last_error()
    assert call(T=5000, x=p + 208, ldx=168, ldbase=168, ldo=168) == 1 and b"workspace" in l.nvfp4_last_error()


# ------------------------------------------------------------------- GPU

SHAPES = [
    (1, 64, 64, 16, 1, 1), (1, 4096, 1000, 16, 3, 1), (2, 8, 1, 16, 2, 1), (7, 72, 33, 32, 3, 1), (64, 512, 768, 64, 9, 1),
    (40, 256, 520, 128, 2, 1), (128, 1000, 333, 48, 40, 3), (100, 136, 64, 96, 1, 100),
    (129, 64, 64, 16, 2, 10), (200, 72, 1, 16, 3, 1), (777, 1000, 203, 48, 9, 37), (300, 520, 264, 128, 5, 20),
    (500, 128, 520, 64, 1, 500), (1000, 8, 96, 32, 300, 1), (5000, 64, 40, 112, 7, 90),
    (256, 64, 72, 32, 60, 1), (257, 64, 72, 32, 60, 1), (300, 4096, 72, 64, 3, 50), (260, 2048, 33, 128, 2, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("T,K,N,r,n,run", SHAPES)
def test_lora(pkg, oracle, cuda, T, K, N, r, n, run, in_place):
    p = Problem(T, K, N, r, n, run)
    a = p.args()
    out = None if in_place else torch.full((T, N), float("nan"), dtype=torch.float16, device=cuda)
    got = pkg.lora_add(*a, out=out)
    torch.cuda.synchronize()
    assert got is (a[0] if in_place else out)
    p.check(oracle, got)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 300])
def test_lora_without_scales_and_ranks(pkg, oracle, cuda, T):
    p = Problem(T, 128, 96, 32, 4, mixed=False)
    p.check(oracle, pkg.lora_add(*p.args()))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [0, 6, 400])
def test_lora_no_tokens_or_no_adapters(pkg, cuda, T):
    p = Problem(T, 64, 72, 16, 2)
    p.adapters[:] = -1
    p.adapters[1::2] = 2          # outside [0, n) as well
    a = p.args()
    out = torch.full_like(a[0], float("nan"))
    pkg.lora_add(*a, out=out)
    assert torch.equal(out, a[0])
    pkg.lora_add(*a)
    assert torch.equal(a[0].cpu(), p.base)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [24, 400])
def test_lora_strides_and_what_lies_around(pkg, oracle, cuda, T):
    """Row and matrix strides, odd output rows, negative ranks (none used),
    ranks beyond r, dirty memory from the allocator."""
    K, N, r, n = 200, 136, 32, 3
    p = Problem(T, K, N, r, n, run=5)
    p.ranks = torch.tensor([32, -3, 99], dtype=torch.int32)
    g = torch.Generator().manual_seed(2)
    p.a = torch.randn((n, r, K), generator=g).div(14).to(torch.float16)
    p.b = torch.randn((n, N, r), generator=g).div(6).to(torch.float16)
    nan = lambda *s: torch.full(s, float("nan"), dtype=torch.float16, device=cuda)
    base, x, a, b, ad, sc, rk = p.args()
    bigx, biga, bigb, bigo = nan(T, K + 24), nan(n + 1, r + 2, K + 8), nan(n, N + 1, r + 16), nan(T + 2, N + 3)
    bigx[:, 8:8 + K], biga[:n, :r, :K], bigb[:, :N, 8:8 + r], bigo[1:T + 1, 1:1 + N] = x, a, b, base
    bigo[[0, T + 1]] = 5
    need = ctypes.c_int64(0)
    pkg._lib.lib().nvfp4_lora_workspace(T, r, n, ctypes.byref(need))
    torch.full((max(need.value, 1),), 0xFF, dtype=torch.uint8, device=cuda)
    got = pkg.lora_add(bigo[1:T + 1, 1:1 + N], bigx[:, 8:8 + K], biga[:n, :r, :K], bigb[:, :N, 8:8 + r], ad, sc, rk)
    p.check(oracle, got)
    assert (bigo[[0, T + 1]] == 5).all() and torch.isnan(bigo[1:T + 1, 0]).all() and torch.isnan(bigo[1:T + 1, N + 1:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [6, 200])
@pytest.mark.parametrize("size", [1e-6, 2e3])
def test_lora_far_ranges(pkg, oracle, cuda, T, size):
    """Inner products far below and above fp16's range, brought back by B: u must not be rounded to fp16."""
    K, N, r, n = 512, 64, 16, 2
    p = Problem(T, K, N, r, n, mixed=False)
    g = torch.Generator().manual_seed(3)
    p.x = (torch.randn((T, K), generator=g) * max(size, 1)).to(torch.float16)
    p.a = (torch.randn((n, r, K), generator=g) * size).to(torch.float16)
    p.b = (torch.randn((n, N, r), generator=g) * (1e-6 if size > 1 else 1e4)).to(torch.float16)
    p.scales = torch.full((n,), 1e-2 if size > 1 else 1.0)      # u * scale is about 1e6, or 2e-5
    p.check(oracle, pkg.lora_add(*p.args()))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [16, 300])
def test_lora_graphs_and_streams(pkg, oracle, cuda, T):
    ps = [Problem(T, 128, 200, 32, 4, seed=s) for s in (1, 2)]
    live = [p.args() for p in ps]
    outs = [torch.empty_like(a[0]) for a in live]
    want = [pkg.lora_add(*a).clone() for a in [p.args() for p in ps]]
    torch.cuda.synchronize()
    graphs = []
    for a, o in zip(live, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            pkg.lora_add(*a, out=o)
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
    live[0][4].copy_(live[1][4])          # other requests through the same graph
    graphs[0].replay()
    torch.cuda.synchronize()
    ps[0].adapters = ps[1].adapters
    ps[0].check(oracle, outs[0])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 300])
def test_lora_calls_at_once_and_column_slices(pkg, oracle, cuda, T):
    """Two eager calls on two streams, and base and x as column slices of one
    buffer."""
    ps = [Problem(T, 256, 192, 32, 4, seed=s) for s in (5, 6)]
    args = [p.args() for p in ps]
    for a in args:
        buf = torch.zeros((T, 256 + 192 + 8), dtype=torch.float16, device=cuda)
        buf[:, :256], buf[:, 256:448] = a[1], a[0]
        a[0], a[1] = buf[:, 256:448], buf[:, :256]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for s, a in zip(streams, args):
        with torch.cuda.stream(s):
            pkg.lora_add(*a)
    torch.cuda.synchronize()
    for p, a in zip(ps, args):
        p.check(oracle, a[0])
    with pytest.raises(RuntimeError, match="overlaps x"):
        pkg.lora_add(args[0][1][:, :192], *args[0][1:])


@pytest.mark.gpu
def test_lora_beside_the_skinny_gemm(pkg, oracle, cuda):
    """The projection as it is used: quantise, shared NVFP4 weights, adapters."""
    T, K, N, r, n = 20, 512, 640, 32, 3
    p = Problem(T, K, N, r, n)
    w = pkg.inputs.operand(N, K, torch.Generator().manual_seed(4), device=cuda)
    base, x, a, b, ad, sc, rk = p.args()
    codes, sf = pkg.quantize(x)
    pkg.skinny_gemm(codes, w.codes, sf, w.sf_blocked, base)
    torch.cuda.synchronize()
    p.base = base.cpu()
    shared = oracle.gemm(codes.cpu(), w.codes.cpu(), sf.cpu(), w.sf_blocked.cpu(), T, N, K)
    np.testing.assert_allclose(p.base.numpy().astype(np.float32), shared, rtol=1e-2, atol=1e-2)
    p.check(oracle, pkg.lora_add(base, x, a, b, ad, sc, rk))


@pytest.mark.gpu
def test_lora_refusals(pkg, cuda):
    p = Problem(4, 64, 72, 16, 2)
    a = p.args()

    def bad(i, t, err, match):
        c = list(a)
        c[i] = t
        with pytest.raises(err, match=match):
            pkg.lora_add(*c)
    bad(0, a[0].cpu(), ValueError, "CUDA")
    bad(0, a[0].float(), TypeError, "float16")
    bad(1, a[1][:3], ValueError, "rows")
    bad(1, a[1].bfloat16(), TypeError, "float16")
    bad(2, a[2][:, :, :32], ValueError, "fit")
    bad(3, a[3][:, :, :8], ValueError, "fit")
    bad(4, a[4].long(), ValueError, "adapters")
    bad(4, a[4][:3], ValueError, "adapters")
    bad(5, a[5].double(), ValueError, "scales")
    bad(6, a[6][:1], ValueError, "ranks")
    with pytest.raises(RuntimeError, match="rank"):
        pkg.lora_add(a[0], a[1], a[2][:, :8].contiguous(), a[3][:, :, :8].contiguous(), a[4])
    with pytest.raises(ValueError, match="out"):
        pkg.lora_add(*a, out=a[0][:3])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 24, 300])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_lora_a_token_that_is_not_finite_stays_alone(pkg, cuda, T, bad):
    p = Problem(T, 128, 96, 32, 3, 7)
    p.adapters[:5] = 0                       # beside others of its adapter, of full rank
    want = pkg.lora_add(*p.args())
    a = list(p.args())
    a[1] = a[1].clone()
    a[1][2] = bad
    got = pkg.lora_add(*a)
    keep = torch.arange(T, device=cuda) != 2
    assert torch.equal(got[keep], want[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N,r,n,run", [
    (2559, 520, 72, 64, 5, 70), (2560, 520, 72, 64, 5, 70), (2600, 1032, 40, 32, 40, 3), (2700, 264, 33, 128, 3, 200),
    (4100, 8, 64, 16, 2, 1000), (9500, 520, 24, 64, 3, 500),
])
def test_lora_both_sides_of_the_rules(pkg, oracle, cuda, T, K, N, r, n, run):
    p = Problem(T, K, N, r, n, run)
    p.check(oracle, pkg.lora_add(*p.args()))


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("T,K,N,r,n", [      # the clusters' sizes for few tokens: 16, 8, 4, 2, 1
    (4, 200, 72, 64, 9), (48, 136, 72, 32, 48), (100, 64, 200, 16, 100), (180, 264, 33, 32, 180), (256, 72, 40, 16, 1000),
    (18, 136, 72, 128, 40), (40, 136, 72, 128, 60), (100, 72, 33, 128, 100), (200, 136, 72, 128, 200), (256, 40, 8, 112, 1),
])
def test_lora_clusters_of_every_size(pkg, oracle, cuda, T, K, N, r, n, in_place):
    p = Problem(T, K, N, r, n)
    a = p.args()
    out = None if in_place else torch.full((T, N), float("nan"), dtype=torch.float16, device=cuda)
    p.check(oracle, pkg.lora_add(*a, out=out))


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N,r,n,run", [     # fewer items than clusters: several share one's columns
    (1, 64, 9000, 16, 2, 1), (1, 200, 8195, 128, 1, 1), (9, 72, 5000, 64, 2, 9), (30, 136, 4104, 32, 200, 30),
    (200, 72, 4099, 16, 900, 200), (256, 40, 2200, 128, 300, 256), (64, 64, 2048, 64, 3, 20),
])
def test_lora_clusters_that_share_an_item(pkg, oracle, cuda, T, K, N, r, n, run):
    p = Problem(T, K, N, r, n, run)
    p.adapters[0] = 0
    for in_place in (False, True):
        a = p.args()
        out = None if in_place else torch.full((T, N), float("nan"), dtype=torch.float16, device=cuda)
        p.check(oracle, pkg.lora_add(*a, out=out))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [6, 300, 2600])
@pytest.mark.parametrize("N", [72, 33])
@pytest.mark.parametrize("r", [16, 64, 128])
@pytest.mark.parametrize("top", [0.3, 300.0])
def test_lora_entries_of_very_different_size(pkg, oracle, cuda, T, N, r, top):
    """A token's inner products from `top` down to 2^-19 of it, each alone in an output column that brings it back.
    An entry keeps 22 bits, or is off by at most 2^-39 of the token's largest; to that come the sum over K in 32 bits (4
    steps of 16 and 24 joined parts, two roundings each), that of the mma's, and fp16's rounding of the result."""
    K, n = 64, 2
    g = torch.Generator().manual_seed(T + N + r)
    size = torch.exp2(-19 * torch.arange(r) / (r - 1))
    x = torch.randn((T, K), generator=g).to(torch.float16)
    a = (torch.randn((n, r, K), generator=g) * (top / K ** 0.5 * size).unsqueeze(1)).to(torch.float16)
    b = torch.zeros((n, N, r))
    alone = torch.arange(N) * (r - 1) // (N - 1)
    b[:, torch.arange(N), alone] = (1 / size[alone]).clamp(max=3e4)
    b = b.to(torch.float16)
    base = torch.zeros((T, N), dtype=torch.float16)
    ad = torch.randint(0, n, (T,), generator=g).to(torch.int32)
    got = pkg.lora_add(*(t.to(cuda) for t in (base, x, a, b, ad))).cpu().double()
    a64, b64, x64 = a.double()[ad.long()], b.double()[ad.long()], x.double()
    u, ua = torch.einsum("trk,tk->tr", a64, x64), torch.einsum("trk,tk->tr", a64.abs(), x64.abs())
    want = torch.einsum("tnr,tr->tn", b64, u)
    eu = (4 + 24) * 2.0 ** -23 * ua + 2.0 ** -22 * u.abs() + 2.0 ** -39 * u.abs().amax(dim=1, keepdim=True)
    tol = torch.einsum("tnr,tr->tn", b64.abs(), eu + (2 * r / 16 + 8) * 2.0 ** -23 * u.abs())
    tol = tol + (want.abs() + tol) * 2.0 ** -11 + 2.0 ** -25
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [300, 2600])
@pytest.mark.parametrize("N,r", [(64, 16), (72, 64), (33, 64), (40, 128), (35, 128)])
@pytest.mark.parametrize("size", [1e-6, 2e3])
def test_lora_far_ranges_of_many_tokens(pkg, oracle, cuda, T, N, r, size):
    """Inner products far below and above fp16's range where two products follow one another, tokens of very different
    size among the rows of one tile, rows of any alignment."""
    K, n = 264, 3
    p = Problem(T, K, N, r, n, run=7, mixed=False)
    g = torch.Generator().manual_seed(3)
    per_token = torch.exp2(-torch.randint(0, 12, (T, 1), generator=g).float())
    p.x = (torch.randn((T, K), generator=g) * max(size, 1) * per_token).to(torch.float16)
    p.a = (torch.randn((n, r, K), generator=g) * size).to(torch.float16)
    p.b = (torch.randn((n, N, r), generator=g) * (1e-6 if size > 1 else 1e4)).to(torch.float16)
    p.scales = torch.full((n,), 1e-2 if size > 1 else 1.0)
    p.check(oracle, pkg.lora_add(*p.args()))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 300])
@pytest.mark.parametrize("N", [72, 33])
def test_lora_rows_without_an_adapter_keep_every_bit(pkg, cuda, T, N):
    """Zeros of both signs, infinities and subnormals of base, where nothing is added: no adapter, or one of rank 0."""
    p = Problem(T, 64, N, 32, 2, mixed=False)
    p.adapters[:] = torch.tensor([-1, 0]).repeat(T)[:T]
    p.ranks = torch.zeros(2, dtype=torch.int32)
    p.base[:, ::3] = -0.0
    p.base[:, 1::5] = float("-inf")
    p.base[:, 2::7] = 6e-8
    a = p.args()
    out = torch.full_like(a[0], 7.0)
    pkg.lora_add(*a, out=out)
    assert torch.equal(out.view(torch.int16), a[0].view(torch.int16))
