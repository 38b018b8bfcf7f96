"""What the Python entry points do before the library, without a GPU: stand-in tensors, and a stand-in library that notes
which device is current when an entry point is called."""
import contextlib
import ctypes
import warnings

import pytest
import torch

FakeTensorMode = pytest.importorskip("torch._subclasses.fake_tensor").FakeTensorMode


class Library:
    def __init__(self, device):
        self.device, self.calls = device, []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, self.device[0]))
            if name == "nvfp4_moe_workspace":
                # as on unlike GPUs: what a call needs depends on the device
                ctypes.cast(args[-1], ctypes.POINTER(ctypes.c_int64))[0] = 1024 * (1 + self.device[0])
            elif name == "nvfp4_moe_mlp":
                return 0 if args[-2] == 1024 * (1 + self.device[0]) else 1
            return 0
        return entry


@pytest.fixture
def two_devices(pkg, monkeypatch):
    current = [0]

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        try:
            yield
        finally:
            current[0] = before
    library = Library(current)
    library.nvfp4_last_error = lambda: b"workspace too small"
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(pkg._lib, "_lib", library)
    monkeypatch.setattr(pkg._lib, "raw_stream", lambda index: index)
    with warnings.catch_warnings(), FakeTensorMode():
        warnings.simplefilter("ignore")              # stand-ins have no address
        yield library


@pytest.mark.parametrize("index", [0, 1])
def test_workspaces_are_asked_for_on_the_tensors_device(pkg, two_devices, index):
    dev, u8 = f"cuda:{index}", torch.uint8
    x = torch.empty((6, 64), dtype=torch.float16, device=dev)
    w = torch.empty((6, 2), dtype=torch.float32, device=dev)
    ids = torch.empty((6, 2), dtype=torch.int32, device=dev)
    codes = torch.empty((4, 64, 32), dtype=u8, device=dev)
    sf = torch.empty((4, pkg.layout.blocked_numel(64, 4)), dtype=u8, device=dev)
    out = pkg.moe_mlp(x, ids, w, codes, codes, codes, sf, sf, sf)
    assert out.device == x.device
    a = torch.empty((2, 16, 64), dtype=torch.float16, device=dev)
    pkg.lora_add(x, x.clone(), a, a.transpose(1, 2).contiguous(), ids[:, 0].contiguous())
    pkg.route_experts(torch.empty((6, 8), device=dev), 2)
    assert [name for name, _ in two_devices.calls] == ["nvfp4_moe_workspace", "nvfp4_moe_mlp", "nvfp4_lora_workspace",
                                                       "nvfp4_lora_add", "nvfp4_route_experts"]
    # the adapters' workspace depends on the sizes alone
    assert {device for name, device in two_devices.calls if name != "nvfp4_lora_workspace"} == {index}


def test_outputs_that_require_a_gradient_are_refused(pkg, two_devices):
    """The library writes behind autograd's back."""
    dev = "cuda:0"
    half = lambda *s: torch.empty(s, dtype=torch.float16, device=dev)
    x, a = half(6, 64), half(2, 16, 64)
    ids = torch.empty((6, 2), dtype=torch.int32, device=dev)
    w = torch.empty((6, 2), dtype=torch.float32, device=dev)
    codes = torch.empty((4, 64, 32), dtype=torch.uint8, device=dev)
    sf = torch.empty((4, pkg.layout.blocked_numel(64, 4)), dtype=torch.uint8, device=dev)
    logits, b, ad = torch.empty((6, 8), device=dev), a.transpose(1, 2).contiguous(), ids[:, 0].contiguous()
    leaf = half(6, 64).requires_grad_()
    projected = leaf * 2                             # what a projection with trained weights returns
    calls = [lambda: pkg.lora_add(projected, x, a, b, ad), lambda: pkg.lora_add(x, x.clone(), a, b, ad, out=projected),
             lambda: pkg.lora_add(leaf, x, a, b, ad),
             lambda: pkg.moe_mlp(x, ids, w, codes, codes, codes, sf, sf, sf, out=projected),
             lambda: pkg.route_experts(logits, 2, weights=torch.empty_like(w).requires_grad_())]
    for call in calls:
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
    assert not any(name in ("nvfp4_lora_add", "nvfp4_moe_mlp", "nvfp4_route_experts") for name, _ in two_devices.calls)
    with torch.no_grad():
        for call in calls:
            call()
    # operands that require one are read, not written
    pkg.lora_add(x, leaf, a.clone().requires_grad_(), b, ad, out=half(6, 64))
