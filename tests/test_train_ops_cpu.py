"""CPU: what the training operators refuse, at the C ABI (every check runs before anything touches a device) and in the
Python binding (tensors that are not on a ROCm device)."""
import ctypes

import pytest
import torch

from f_lite import _native as nat


@pytest.fixture(scope="module")
def lib():
    import build_native

    build_native.build(verbose=False)
    return nat.load()


PTR = 1 << 20  # an aligned address that no refused call reads


def attn_args(**kw):
    a = nat.AttnTrain()
    for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv", "cu_q", "cu_k"):
        setattr(a, n, PTR)
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        setattr(a, n + "_row", 4 * 64)
        setattr(a, n + "_head", 64)
    a.batch, a.heads, a.kv_heads, a.head_dim, a.total_q, a.total_k, a.scale = 1, 4, 2, 64, 10, 10, 0.125
    for n, v in kw.items():
        setattr(a, n, v)
    return a


BAD_ATTN = [
    (dict(head_dim=96), b"head size"), (dict(head_dim=0), b"head size"), (dict(batch=0), b"positive"),
    (dict(heads=3), b"multiple of kv heads"), (dict(kv_heads=0), b"positive"), (dict(heads=-4), b"positive"),
    (dict(total_q=-1), b"negative"), (dict(cu_q=None), b"cu_seqlens"), (dict(cu_k=None), b"cu_seqlens"),
    (dict(heads=1 << 27, kv_heads=1), b"too many"), (dict(q=None), b"missing q"), (dict(k=None), b"missing k"),
    (dict(v=None), b"missing v"), (dict(out=None), b"missing out"), (dict(lse=None), b"missing lse"),
    (dict(q=PTR + 2), b"q must be"), (dict(k_row=260), b"k must be"), (dict(v_head=60), b"v must be"),
    (dict(out_row=32), b"out must be"), (dict(q_row=(1 << 22) + 8), b"q must be"),
]
BAD_ATTN_BWD = [(dict(dout=None), b"missing dout"), (dict(dq=None), b"missing dq"), (dict(dk=None), b"missing dk"),
                (dict(dv=None), b"missing dv"), (dict(dout_row=4), b"dout must be"), (dict(dk=PTR + 8), b"dk must be")]


@pytest.mark.parametrize("kw,msg", BAD_ATTN)
def test_attention_forward_refuses(lib, kw, msg):
    assert lib.flite_attn_lse_fwd(None, ctypes.byref(attn_args(**kw)), PTR, 1 << 40) != 0
    assert msg in lib.flite_last_error()


@pytest.mark.parametrize("kw,msg", BAD_ATTN + BAD_ATTN_BWD)
def test_attention_backward_refuses(lib, kw, msg):
    assert lib.flite_attn_lse_bwd(None, ctypes.byref(attn_args(**kw)), PTR, 1 << 40) != 0
    assert msg in lib.flite_last_error()


def test_attention_workspace(lib):
    n = lib.flite_attn_lse_bwd_workspace_bytes(ctypes.byref(attn_args()))
    assert n >= 4 * 10 * 8
    for ws, size in ((None, 1 << 40), (PTR, n - 1), (PTR + 16, 1 << 40)):
        assert lib.flite_attn_lse_bwd(None, ctypes.byref(attn_args()), ws, size) != 0
        assert b"workspace" in lib.flite_last_error()
    assert lib.flite_attn_lse_bwd_workspace_bytes(ctypes.byref(attn_args(head_dim=80))) == -1
    assert lib.flite_attn_lse_bwd_workspace_bytes(None) == -1
    assert lib.flite_attn_lse_fwd_workspace_bytes(None) == -1
    # one query over many keys: the sweep is cut
    long_sweep = attn_args(total_q=1, total_k=8192)
    n = lib.flite_attn_lse_fwd_workspace_bytes(ctypes.byref(long_sweep))
    assert n > 0
    for ws, size in ((None, 1 << 40), (PTR, n - 1), (PTR + 16, 1 << 40)):
        assert lib.flite_attn_lse_fwd(None, ctypes.byref(long_sweep), ws, size) != 0
        assert b"workspace" in lib.flite_last_error()
    assert lib.flite_attn_lse_fwd(None, None, None, 0) != 0 and lib.flite_attn_lse_bwd(None, None, None, 0) != 0


def rope_args(**kw):
    a = nat.RopeAxesArgs()
    a.x = a.out = a.y = a.rstd = a.positions = PTR
    pairs, bases = kw.pop("pairs", (8, 12, 12)), kw.pop("bases", (1e4, 1e4, 1e4))
    a.axis_pairs, a.bases = (ctypes.c_int * 8)(*pairs[:8]), (ctypes.c_double * 8)(*bases[:8])
    a.x_row = a.out_row = a.y_row = 256
    a.x_head = a.out_head = a.y_head = 64
    a.rows, a.tokens, a.axes, a.heads, a.rope_heads, a.head_dim = 10, 5, len(pairs), 4, 4, 64
    a.is_bf16, a.norm, a.eps = 1, 1, 1e-6
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(head_dim=72), b"head size"), (dict(head_dim=272), b"head size"), (dict(axes=0), b"axes"),
    (dict(pairs=(8,) * 9, bases=(1e4,) * 9), b"axes"), (dict(pairs=(8, 12, 13)), b"more pairs"),
    (dict(pairs=(8, 12, 11)), b"multiple of 8"), (dict(pairs=(-8, 16, 16)), b"more pairs"),
    (dict(pairs=(0, 0, 0)), b"multiple of 8"), (dict(bases=(1e4, 0.0, 1e4)), b"bases"),
    (dict(bases=(1e4, float("nan"), 1e4)), b"bases"), (dict(bases=(1e4, float("inf"), 1e4)), b"bases"),
    (dict(rows=-1), b"rows"), (dict(heads=0), b"heads"), (dict(rope_heads=5), b"rope_heads"),
    (dict(positions=None), b"positions"), (dict(tokens=0), b"positions"), (dict(x=None), b"aligned"),
    (dict(out=PTR + 4), b"aligned"), (dict(x_row=260), b"aligned"), (dict(out_head=36), b"aligned"),
    (dict(rstd=None), b"rstd"),
])
def test_rope_axes_refuses(lib, kw, msg):
    for f in (lib.flite_rope_axes_fwd, lib.flite_rope_axes_bwd):
        assert f(None, ctypes.byref(rope_args(**dict(kw)))) != 0
        assert msg in lib.flite_last_error()


def test_rope_axes_backward_needs_the_output(lib):
    for kw in (dict(y=None), dict(y=PTR + 2), dict(y_row=4)):
        assert lib.flite_rope_axes_bwd(None, ctypes.byref(rope_args(**kw))) != 0
        assert b"output" in lib.flite_last_error()
    assert lib.flite_rope_axes_fwd(None, None) != 0


def norm_args(**kw):
    a = nat.NormArgs()
    for n in ("x", "y", "dy", "dx", "w", "b", "shift", "scale", "dw", "db", "dshift", "dscale"):
        setattr(a, n, PTR)
    a.ldx = a.ldy = a.lddy = a.lddx = a.mod_seg_stride = a.dim = 64
    a.rows, a.seg_rows, a.eps = 10, 4, 1e-6
    for n, v in kw.items():
        setattr(a, n, v)
    return a


BAD_NORM = [(dict(dim=60), b"dim"), (dict(dim=0), b"dim"), (dict(dim=8200, ldx=8200), b"dim"), (dict(rows=-1), b"rows"),
            (dict(seg_rows=-1), b"seg_rows"), (dict(x=None), b"x must be"), (dict(ldx=56), b"x must be"),
            (dict(ldx=68), b"x must be"), (dict(w=PTR + 2), b"w and b"), (dict(scale=PTR + 4), b"shift and scale"),
            (dict(mod_seg_stride=66), b"shift and scale")]


@pytest.mark.parametrize("kw,msg", BAD_NORM + [(dict(y=None), b"y must be"), (dict(ldy=32), b"y must be"),
                                               (dict(rms=1), b"rmsnorm_modulate")])
def test_layernorm_refuses(lib, kw, msg):
    assert lib.flite_layernorm_modulate(None, ctypes.byref(norm_args(**kw))) != 0
    assert msg in lib.flite_last_error()


@pytest.mark.parametrize("kw,msg", BAD_NORM + [
    (dict(dy=None), b"dy must be"), (dict(lddy=4), b"dy must be"), (dict(dx=PTR + 8), b"dx must be"),
    (dict(rms=1), b"no bias"), (dict(w=None), b"not given"), (dict(b=None), b"not given"),
    (dict(scale=None), b"not given")])
def test_norm_backward_refuses(lib, kw, msg):
    assert lib.flite_norm_modulate_bwd(None, ctypes.byref(norm_args(**kw)), PTR, 1 << 40) != 0
    assert msg in lib.flite_last_error()


def test_norm_workspace(lib):
    n = lib.flite_norm_bwd_workspace_bytes(10, 4, 64)
    assert n >= 3 * 2 * 64 * 4  # S0 and S1 of three segments
    for ws, size in ((None, 1 << 40), (PTR, n - 1), (PTR + 4, 1 << 40)):
        assert lib.flite_norm_modulate_bwd(None, ctypes.byref(norm_args()), ws, size) != 0
        assert b"workspace" in lib.flite_last_error()
    assert lib.flite_norm_bwd_workspace_bytes(0, 0, 64) == 0
    assert lib.flite_norm_modulate_bwd(None, None, None, 0) != 0


def test_python_refuses_cpu_tensors():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    x = torch.zeros(4, 64)
    pos = torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: nat.attn_varlen_lse(q, q, q, cu, cu, 0.1),
                 lambda: nat.attn_varlen_bwd(q, q, q, q, q, torch.zeros(2, 4), cu, cu, 0.1),
                 lambda: nat.rope_axes(q, pos, (16, 16)), lambda: nat.rope_axes_bwd(q, pos, (16, 16)),
                 lambda: nat.layernorm_modulate(x), lambda: nat.norm_modulate_bwd(x.bfloat16(), x)):
        with pytest.raises(nat.FliteError, match="ROCm device"):
            call()
