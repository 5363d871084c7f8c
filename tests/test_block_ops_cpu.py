"""No-GPU checks of cross attention and of the q/k norm with rotation: structure layouts, argument
validation of the C entry points before any launch, refusals of the operators, routing of the mode."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

import paraattention_b200 as pa
from paraattention_b200 import _lib as L
from paraattention_b200 import build_ext, config, ops

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def lib():
    build_ext.build()
    return L.load()


def test_struct_layouts_match_c(tmp_path):
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pa_b200.h"\n'
                   'int main(){printf("%zu %zu %zu %zu\\n", sizeof(pa_xattn_args), offsetof(pa_xattn_args, key_mask),'
                   ' offsetof(pa_xattn_args, q_stride), offsetof(pa_xattn_args, workspace_bytes));'
                   'printf("%zu %zu %zu\\n", sizeof(pa_qk_norm_args), offsetof(pa_qk_norm_args, cos),'
                   ' offsetof(pa_qk_norm_args, workspace));}\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(L.XattnArgs), L.XattnArgs.key_mask.offset, L.XattnArgs.q_stride.offset,
                   L.XattnArgs.workspace_bytes.offset, C.sizeof(L.QkNormArgs), L.QkNormArgs.cos.offset,
                   L.QkNormArgs.workspace.offset]


def _xattn(addr):
    a = L.XattnArgs()
    for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv"):
        setattr(a, n, addr)
    a.batch = a.kv_batch = 2
    a.heads, a.kv_heads, a.seq_q, a.seq_kv, a.head_dim, a.scale = 4, 2, 300, 77, 64, 0.125
    for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
        getattr(a, n + "_stride")[:] = (64 * 4 * 300, 64, 64 * 4)
    return a


def test_cross_attention_validates_before_any_launch(lib):
    buf = (C.c_uint8 * 256)()
    addr = (C.addressof(buf) + 15) // 16 * 16
    assert lib.pa_xattn_fwd(None, None) == L.PA_EINVAL and lib.pa_xattn_bwd(None, None) == L.PA_EINVAL
    for field, value in (("batch", 0), ("heads", 0), ("kv_heads", 3), ("seq_q", 0), ("seq_kv", 0), ("kv_batch", 3),
                         ("dtype", 2), ("scale", 0.0), ("scale", float("nan")), ("scale", float("inf")), ("q", None),
                         ("k", None), ("v", None), ("out", None), ("q", addr + 2), ("seq_q", 2000000000)):
        a = _xattn(addr)
        setattr(a, field, value)
        for fn in (lib.pa_xattn_fwd, lib.pa_xattn_bwd):
            assert fn(C.byref(a), None) == L.PA_EINVAL, (field, value)
    a = _xattn(addr)
    a.head_dim = 96
    assert lib.pa_xattn_fwd(C.byref(a), None) == L.PA_ENOTSUP
    assert lib.pa_xattn_workspace_bytes(C.byref(a), 0) == L.PA_ENOTSUP
    a = _xattn(addr)
    a.k_stride[2] = 65
    assert lib.pa_xattn_fwd(C.byref(a), None) == L.PA_EINVAL
    for field in ("lse", "dout", "dq", "dk", "dv"):
        a = _xattn(addr)
        setattr(a, field, None)
        assert lib.pa_xattn_bwd(C.byref(a), None) == L.PA_EINVAL, field
    # a workspace that is missing, too small or misaligned
    a = _xattn(addr)
    n = lib.pa_xattn_workspace_bytes(C.byref(a), 1)
    assert n >= 2 * 4 * 384 * 8
    assert lib.pa_xattn_bwd(C.byref(a), None) == L.PA_EINVAL and b"workspace" in lib.pa_last_error()
    a.workspace, a.workspace_bytes = addr // 256 * 256 + 256, n - 1
    assert lib.pa_xattn_bwd(C.byref(a), None) == L.PA_EINVAL
    a.workspace, a.workspace_bytes = addr // 256 * 256 + 16, n
    assert lib.pa_xattn_bwd(C.byref(a), None) == L.PA_EINVAL


def test_cross_attention_backward_of_one_side(lib):
    """dq alone and dk with dv get as far as the missing workspace; nothing at all, or half a pair, do not."""
    buf = (C.c_uint8 * 256)()
    addr = (C.addressof(buf) + 15) // 16 * 16
    for gone, what in ((("dq",), b"workspace"), (("dk", "dv"), b"workspace"), (("dq", "dk", "dv"), b"computes"),
                       (("dk",), b"computes"), (("dv",), b"dv"), (("dq", "dv"), b"dv")):
        a = _xattn(addr)
        for field in gone:
            setattr(a, field, None)
        assert lib.pa_xattn_bwd(C.byref(a), None) == L.PA_EINVAL and what in lib.pa_last_error(), gone


def test_cross_attention_workspace_sizes(lib):
    a = _xattn(0)
    assert lib.pa_xattn_workspace_bytes(C.byref(a), 0) == 0  # few tiles of keys: nothing to divide
    a.key_mask = 16
    masked = lib.pa_xattn_workspace_bytes(C.byref(a), 0)
    assert masked == 256 + 256  # 2 x 2 words of 64 keys, 2 extents
    a = _xattn(0)
    a.seq_kv = 50000  # few units, many tiles: partial results of two slots per CTA
    assert lib.pa_xattn_workspace_bytes(C.byref(a), 0) >= 2 * 256 * (64 + 2) * 4
    a.seq_q = 2  # few rows: joined in shared memory
    assert lib.pa_xattn_workspace_bytes(C.byref(a), 0) == 0


def test_qk_norm_validates_before_any_launch(lib):
    buf = (C.c_uint8 * 256)()
    addr = (C.addressof(buf) + 15) // 16 * 16

    def args():
        a = L.QkNormArgs()
        for i in range(2):
            a.x[i] = a.y[i] = a.dy[i] = a.weight[i] = a.dweight[i] = addr
            for s in (a.x_stride, a.y_stride, a.dy_stride):
                s[i][:] = (640, 128, 64)
        a.heads[:] = (2, 1)
        a.batch, a.rows, a.head_dim, a.eps, a.interleaved = 1, 5, 64, 1e-6, 1
        return a

    assert lib.pa_qk_norm_fwd(None, None) == L.PA_EINVAL
    for field, value in (("batch", 0), ("rows", 0), ("dtype", 5), ("eps", -1.0), ("eps", float("nan")), ("cos", addr),
                         ("table_row0", -1)):
        a = args()
        setattr(a, field, value)
        assert lib.pa_qk_norm_fwd(C.byref(a), None) == L.PA_EINVAL, field
    a = args()
    a.head_dim = 80
    assert lib.pa_qk_norm_fwd(C.byref(a), None) == L.PA_ENOTSUP
    for change in (lambda a: a.x.__setitem__(0, None), lambda a: a.y.__setitem__(1, None), lambda a: a.x.__setitem__(1, addr + 2),
                   lambda a: a.heads.__setitem__(1, 0), lambda a: a.x_stride[0].__setitem__(1, 4), lambda a: a.weight.__setitem__(0, addr + 8)):
        a = args()
        change(a)
        assert lib.pa_qk_norm_fwd(C.byref(a), None) == L.PA_EINVAL
    a = args()
    assert lib.pa_qk_norm_bwd(C.byref(a), None) == L.PA_EINVAL and b"workspace" in lib.pa_last_error()
    a.dy[0] = None
    assert lib.pa_qk_norm_bwd(C.byref(a), None) == L.PA_EINVAL
    assert lib.pa_qk_norm_workspace_bytes() > 0


def test_operators_refuse_cpu_tensors():
    q = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="CUDA"):
        ops.cross_attention(q, q, q)
    with pytest.raises(AssertionError, match="CUDA"):
        ops.qk_norm_rotary(q, q)
    with pytest.raises(AssertionError, match="CUDA"):
        pa.cross_attn_func(q, q[:, :, :3], q[:, :, :3])


def test_cross_attn_func_refuses_what_it_does_not_compute():
    q, k = torch.zeros(2, 4, 8, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 5, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="dropout"):
        pa.cross_attn_func(q, q, q, dropout_p=0.1)
    with pytest.raises(NotImplementedError, match="is_causal"):
        pa.cross_attn_func(q, q, q, is_causal=True)
    with pytest.raises(AssertionError, match="enable_gqa"):
        pa.cross_attn_func(q, k, k)
    for mask in (torch.zeros(2, 1, 8, 5), torch.ones(2, 1, 8, 5, dtype=torch.bool), torch.zeros(2, 1, 1, 5)):
        with pytest.raises(NotImplementedError, match="key-padding"):
            pa.cross_attn_func(q, k, k, mask, enable_gqa=True)


def test_cross_attn_mode_takes_the_calls_with_other_lengths():
    from paraattention_b200 import para_attn_interface as I

    seen = []
    real = I.cross_attn_func
    I.cross_attn_func = lambda *a, **k: seen.append((a[0].shape[-2], a[1].shape[-2], k.get("scale"))) or a[0]
    try:
        q, k = torch.randn(1, 2, 8, 64), torch.randn(1, 2, 5, 64)
        want = F.scaled_dot_product_attention(q, q, q)
        with pa.CrossAttnMode():
            assert torch.equal(F.scaled_dot_product_attention(q, q, q), want) and not seen
            F.scaled_dot_product_attention(q, k, k, scale=0.5)
            assert seen == [(8, 5, 0.5)]
            with pa.CrossAttnMode.disable():
                F.scaled_dot_product_attention(q, k, k)
            assert len(seen) == 1
        with pa.CrossAttnMode(same_length=True):
            F.scaled_dot_product_attention(q, q, q)
        assert seen[-1][:2] == (8, 8)
        # a context-parallel mode that skips short keys hands them on
        with pa.CrossAttnMode():
            mode = pa.UnifiedAttnMode.__new__(pa.UnifiedAttnMode)
            mode._skip_small_kv = True
            F.scaled_dot_product_attention(q, k, k)
            n = len(seen)
            out = mode.__torch_function__(F.scaled_dot_product_attention, (), (q, k, k), {})
            assert len(seen) == n + 1 and out is q
    finally:
        I.cross_attn_func = real


def test_differentiable_preparation_is_off_by_default():
    assert config.attention.differentiable is False
