"""Routing, experts' MLP and adapters on inputs and outputs of more than 2^31 elements: rows from both ends and the middle
against the same rows in a call of their own.  A row's arithmetic depends on neither its place nor its neighbours, but
the forms for few and many tokens round differently: the experts' MLP is called at a size of the same form, the adapters
are compared with the oracle."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _some(T, n=40):
    return torch.unique(torch.cat([torch.arange(n), torch.arange(T // 2, T // 2 + n), torch.arange(T - n, T)]))


def test_route_long(pkg, oracle, cuda):
    T, E, k = 8_600_000, 256, 8
    assert T * E > 1 << 31
    x = torch.empty((T, E), dtype=torch.bfloat16, device=cuda).normal_(generator=torch.Generator(cuda).manual_seed(1))
    w, ids = pkg.route_experts(x, k, score="sigmoid", num_groups=8, top_groups=4)
    rows = _some(T).to(cuda)
    rw, ri = oracle.route(x[rows], k, score="sigmoid", groups=8, top_groups=4)
    np.testing.assert_array_equal(ids[rows].cpu().numpy(), ri)
    np.testing.assert_allclose(w[rows].cpu().numpy().astype(np.float64), rw, rtol=6e-6)


def test_lora_long(pkg, oracle, cuda):
    T, K, N, r, n = 200_000, 64, 11_008, 16, 3
    assert T * N > 1 << 31
    g = torch.Generator(cuda).manual_seed(2)
    base = torch.empty((T, N), dtype=torch.float16, device=cuda).normal_(generator=g)
    x = torch.empty((T, K), dtype=torch.float16, device=cuda).normal_(generator=g)
    a = torch.empty((n, r, K), dtype=torch.float16, device=cuda).normal_(generator=g)
    b = torch.empty((n, N, r), dtype=torch.float16, device=cuda).normal_(generator=g)
    ad = torch.randint(-1, n, (T,), device=cuda, generator=g, dtype=torch.int32)
    rows = _some(T).to(cuda)
    want, tol = oracle.lora_add(base[rows], x[rows], a, b, ad[rows])
    got = pkg.lora_add(base, x, a, b, ad)[rows].cpu().double().numpy()
    assert (np.abs(got - want) <= tol).all()


def test_lora_few_tokens_far_apart(pkg, oracle, cuda):
    """Row and matrix strides whose products pass 2^31 elements, in the one-launch form."""
    T, K, N, r, n = 9, 64, 72, 16, 3
    g = torch.Generator(cuda).manual_seed(3)
    room = torch.zeros(2 * (1 << 31) + (1 << 20), dtype=torch.float16, device=cuda)
    far = (1 << 31) // (T - 2) // 8 * 8
    step = 3 * (1 << 29)
    take = lambda shape, strides, at: room.as_strided(shape, strides, at)
    base, x = take((T, N), (far, 1), 0), take((T, K), (far, 1), 1024)
    a, b = take((n, r, K), (step, K, 1), 8192), take((n, N, r), (step, r, 1), 65536)
    for t in (base, x, a, b):
        t.copy_(torch.empty(t.shape, device=cuda).normal_(generator=g))
    ad = torch.tensor([0, 1, 2, -1, 2, 1, 0, 2, 2], dtype=torch.int32, device=cuda)
    want, tol = oracle.lora_add(base, x, a, b, ad)
    out = torch.empty((T, N), dtype=torch.float16, device=cuda)
    pkg.lora_add(base, x, a, b, ad, out=out)
    assert (np.abs(out.cpu().double().numpy() - want) <= tol).all()
    pkg.lora_add(base, x, a, b, ad)
    assert torch.equal(base, out)


def test_moe_long(pkg, cuda):
    T, k, E, D, F = 530_000, 1, 2, 4096, 128
    assert T * D > 1 << 31
    g = torch.Generator(cuda).manual_seed(4)
    x = torch.empty((T, D), dtype=torch.float16, device=cuda).normal_(generator=g)
    ids = torch.randint(-1, E, (T, k), device=cuda, generator=g, dtype=torch.int32)
    w = torch.rand((T, k), device=cuda, generator=g)
    byte = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device=cuda, dtype=torch.uint8)
    rest = [byte(0, 256, E, F, D // 2), byte(0, 256, E, F, D // 2), byte(0, 256, E, D, F // 2)]
    rest += [byte(2, 11, E, pkg.layout.blocked_numel(rows, K // 16)) for rows, K in ((F, D), (F, D), (D, F))]
    rows = _some(T, 300).to(cuda)
    got = pkg.moe_mlp(x, ids, w, *rest)[rows]
    want = pkg.moe_mlp(x[rows], ids[rows], w[rows], *rest)
    assert torch.equal(got, want) and pkg._lib.device_errors() == 0
