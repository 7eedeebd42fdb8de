"""Refusals of the products' entries that need no GPU, and the layout of their C struct."""
import ctypes
import os
import subprocess

import pytest
import torch

from tests.conftest import ROOT


def test_struct_layout_matches_the_header(tmp_path):
    from object_detection_amd.layers import Product
    fields = [n for n, _ in Product._fields_]
    src = tmp_path / "layout.c"
    prints = "".join(f'printf("{n} %zu\\n", offsetof(dh_product, {n}));' for n in fields)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dethead.h"\n'
                   f'int main(void) {{ printf("size %zu\\n", sizeof(dh_product)); {prints} return 0; }}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(Product)
    for n in fields:
        assert int(got[n]) == getattr(Product, n).offset, n


def test_no_cpu_path():
    from object_detection_amd.layers import head_convs, linear, pointwise_conv
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    for call in (lambda: linear(x, w), lambda: pointwise_conv(x.view(1, 8, 2, 2), w), lambda: head_convs([x.view(1, 8, 2, 2)], [w], [None])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(ValueError, match="activation"):
        linear(x, w, activation="tanh")
    with pytest.raises(TypeError):
        linear(None, w)


def test_entry_refuses_bad_arguments():
    """Argument errors come back before anything is launched, so they need no GPU (addresses are never read)."""
    from object_detection_amd import _lib as L
    from object_detection_amd.layers import Product
    lib = L.lib()

    def call(n=1, dtype=0, act=0, ws=None, ws_bytes=0, **changes):
        good = dict(a=4096, b=8192, out=16384, lda=64, ldb=64, ldo=64, I=64, J=64, R=64, batch=1, a_by_reduction=1, b_by_reduction=1)
        p = (Product * max(n, 1))(*[Product(**(good | changes))] * max(n, 1))
        return lib.dh_products(p, n, dtype, act, ws, ws_bytes, None)
    assert call(n=0) == -1 and call(n=6) == -1
    assert call(dtype=3) == -1 and call(dtype=-1) == -1
    assert call(act=5) == -1 and call(act=-1) == -1
    assert call(out=0) == -1 and call(a=0) == -1 and call(b=0) == -1
    assert call(I=-1) == -1 and call(J=-1) == -1 and call(R=-1) == -1 and call(batch=-1) == -1
    assert call(lda=-1) == -1 and call(ldo=-4) == -1
    assert call(a_by_reduction=0) == -1
    assert call(a_batch=-1) == -1 and call(res_batch=-8) == -1
    assert call(I=(1 << 31) - 1) == -1 and call(R=(1 << 31) - 512) == -1
    assert call(a_sum=4096, batch=2) == -1 and call(a_sum=4096, J=0) == -1
    assert call(a=4098) == -3 and call(dtype=1, out=16385) == -3
    assert call(R=1 << 16, lda=1 << 16, ldb=1 << 16) == -4                      # a split reduction needs its workspace
    assert call(I=1 << 30, J=1 << 30) == -1                                     # more tiles than a launch has
    assert lib.dh_products(None, 1, 0, 0, None, 0, None) == -1
    assert lib.dh_products_workspace(None, 1, 0) == 0
    assert lib.dh_product_slope(None, None, None, None, -1, 8, 8, 0, 0, None, 0, None) == -1
    assert lib.dh_product_slope(4096, 4096, None, None, 8, 8, 8, 2, 0, None, 0, None) == -1
    assert lib.dh_product_slope(4096, None, None, 4096, 8, 8, 8, 0, 0, None, 0, None) == -4
    assert lib.dh_product_slope(4096, None, None, 4096, 8, 8, 8, 9, 0, None, 0, None) == -1
    assert lib.dh_product_slope(4098, None, None, 4096, 8, 8, 8, 0, 0, 8192, 1 << 20, None) == -3


def test_detect_with_fused_convolutions_on_the_cpu():
    """The pass on the CPU that derives a model's strides goes through the layers themselves."""
    from object_detection_amd.yolo import Detect
    det = Detect(3, [[1, 2, 3, 4]], (4,))
    det.fused_convs = True
    det.train()
    assert det([torch.zeros(1, 4, 5, 6)])[0].shape == (1, 2, 5, 6, 8)


def test_which_layers_the_fused_head_replaces():
    from object_detection_amd.yolo import _plain_conv
    nn = torch.nn
    assert _plain_conv(nn.Conv2d(4, 6, 1)) and _plain_conv(nn.Conv2d(4, 6, 1, bias=False))
    for m in (nn.Conv2d(4, 6, 3), nn.Conv2d(4, 6, 1, stride=2), nn.Conv2d(4, 6, 1, padding=1), nn.Conv2d(4, 6, 1, groups=2),
              nn.Sequential(nn.Conv2d(4, 6, 1))):
        assert not _plain_conv(m)
    for hook in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"):
        m = nn.Conv2d(4, 6, 1)
        handle = getattr(m, hook)(lambda *a: None)
        assert not _plain_conv(m)
        handle.remove()
        assert _plain_conv(m)


def test_slope_entry_refuses_extents_whose_product_leaves_64_bits():
    from object_detection_amd import _lib as L
    far = 1 << 39
    for z in (None, 4096):
        assert L.lib().dh_product_slope(None, z, None, 4096, far, 1 << 20, far, 2, 0, 8192, 1 << 40, None) == -1
    assert L.lib().dh_product_slope(None, None, None, 4096, far, 1 << 23, 1, 0, 0, 8192, 1 << 40, None) == -1


def test_slope_entry_has_nothing_to_launch_without_elements():
    """No rows, or maps without cells, and no bias gradient wanted: the call ends on the host, whatever the addresses."""
    from object_detection_amd import _lib as L
    for outer, inner in ((0, 1), (0, 7), (2, 0), (0, 0)):
        for at in (None, 4096):
            assert L.lib().dh_product_slope(at, 4096, at, None, outer, 8, inner, 2, 0, None, 0, None) == 0


def test_a_fused_head_keeps_what_torch_would_call():
    """Hooks of all modules, a forward, a convolution or a call that an instance brings along: the layer itself runs."""
    from object_detection_amd.yolo import _plain_conv
    nn, module = torch.nn, torch.nn.modules.module
    m = nn.Conv2d(4, 6, 1)
    for register in (module.register_module_forward_hook, module.register_module_forward_pre_hook, module.register_module_full_backward_hook,
                     module.register_module_full_backward_pre_hook):
        handle = register(lambda *a: None)
        try:
            assert not _plain_conv(m)
        finally:
            handle.remove()
        assert _plain_conv(m)
    for name in ("forward", "_conv_forward"):
        m = nn.Conv2d(4, 6, 1)
        setattr(m, name, lambda *a: None)
        assert not _plain_conv(m)
        delattr(m, name)
        assert _plain_conv(m)
    m = nn.Conv2d(4, 6, 1)
    m.compile()
    assert not _plain_conv(m)
    for make in (nn.utils.parametrizations.weight_norm, nn.utils.parametrizations.spectral_norm):
        assert not _plain_conv(make(nn.Conv2d(4, 6, 1)))


def test_the_number_of_levels_is_the_header_s():
    from object_detection_amd.layers import MAX_LEVELS
    with open(os.path.join(ROOT, "include", "dethead.h")) as f:
        assert f"#define DH_MAX_PRODUCTS {MAX_LEVELS}\n" in f.read()
