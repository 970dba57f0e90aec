"""Refusals and host-side rules of group_norm_act, dropout_act and dense_act that need no GPU."""

import ctypes
import os
import subprocess

import pytest
import torch

from selectssm_b200 import _lib, block_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_header(tmp_path):
    pairs = [("ssm_dropout_params_t", _lib.SSMDropoutParams), ("ssm_group_norm_params_t", _lib.SSMGroupNormParams),
             ("ssm_dense_params_t", _lib.SSMDenseParams)]
    body = ""
    for i, (c, cls) in enumerate(pairs):
        body += "".join(f'printf("{i} {f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in cls._fields_)
        body += f'printf("{i} - %zu\\n", sizeof({c}));'
    src, exe = tmp_path / "lay.c", tmp_path / "lay"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "selectssm_b200.h"\nint main(){' + body + "}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        i, field, value = line.split()
        cls = pairs[int(i)][1]
        assert int(value) == (ctypes.sizeof(cls) if field == "-" else getattr(cls, field).offset), line


def test_abi_refusals_without_gpu():
    lib = _lib.load()
    p = _lib.SSMDropoutParams()
    p.rows, p.dim, p.drop = 2, 0, 0
    assert lib.ssm_dropout_act_fwd(ctypes.byref(p), None) == _lib.SSM_ERR_SHAPE
    p.dim, p.drop = 8, 65537
    assert lib.ssm_dropout_act_fwd(ctypes.byref(p), None) == _lib.SSM_ERR_SHAPE
    p.drop, p.x_stride = 100, 4
    assert lib.ssm_dropout_act_bwd(ctypes.byref(p), None) == _lib.SSM_ERR_SHAPE
    p.x_stride, p.dtype = 0, 9
    assert lib.ssm_dropout_act_fwd(ctypes.byref(p), None) == _lib.SSM_ERR_DTYPE
    p.dtype, p.act = 0, 4
    assert lib.ssm_dropout_act_fwd(ctypes.byref(p), None) == _lib.SSM_ERR_SHAPE
    p.act = 0
    assert lib.ssm_dropout_act_fwd(ctypes.byref(p), None) == _lib.SSM_ERR_NULL
    assert lib.ssm_dropout_act_bwd(None, None) == _lib.SSM_ERR_NULL
    p.rows = 0
    assert lib.ssm_dropout_act_fwd(ctypes.byref(p), None) == _lib.SSM_OK

    g = _lib.SSMGroupNormParams()
    g.batch, g.seqlen, g.dim, g.groups = 2, 5, 30, 4
    assert lib.ssm_group_norm_act_fwd(ctypes.byref(g), None) == _lib.SSM_ERR_SHAPE
    g.groups = 3
    assert lib.ssm_group_norm_act_fwd(ctypes.byref(g), None) == _lib.SSM_ERR_NULL
    g.dtype = 5
    assert lib.ssm_group_norm_act_bwd(ctypes.byref(g), None) == _lib.SSM_ERR_DTYPE
    g.dtype = 0
    g.x = g.y = g.dy = g.dx = g.stats = 0x1000
    need = lib.ssm_group_norm_bwd_workspace_bytes(ctypes.byref(g))
    assert need > 0
    g.workspace, g.workspace_bytes = 0x1000, need - 1
    assert lib.ssm_group_norm_act_bwd(ctypes.byref(g), None) == _lib.SSM_ERR_WORKSPACE
    g.dim = g.groups = 32
    g.x = 0x1004
    assert lib.ssm_group_norm_act_fwd(ctypes.byref(g), None) == _lib.SSM_ERR_ALIGN

    d = _lib.SSMDenseParams()
    d.rows, d.fin, d.fout = 4, 0, 8
    assert lib.ssm_dense_act_fwd(ctypes.byref(d), None) == _lib.SSM_ERR_SHAPE
    d.fin, d.res_stride = 8, 7
    assert lib.ssm_dense_act_fwd(ctypes.byref(d), None) == _lib.SSM_ERR_SHAPE
    d.res_stride, d.dkernel_dtype = 0, 3
    assert lib.ssm_dense_act_bwd(ctypes.byref(d), None) == _lib.SSM_ERR_DTYPE
    d.dkernel_dtype = 0
    assert lib.ssm_dense_act_fwd(ctypes.byref(d), None) == _lib.SSM_ERR_NULL
    d.dy, d.act = 0x1000, 1
    assert lib.ssm_dense_act_bwd(ctypes.byref(d), None) == _lib.SSM_ERR_NULL  # needs pre
    d.act = 0
    assert lib.ssm_dense_act_bwd(ctypes.byref(d), None) == _lib.SSM_ERR_WORKSPACE


def test_python_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        block_ops.dropout_act(x, 0.5, (1, 2))
    with pytest.raises(ValueError, match="CUDA"):
        block_ops.group_norm_act(x, groups=4)
    with pytest.raises(ValueError, match="CUDA"):
        block_ops.dense_act(x, torch.zeros(8, 8))
    with pytest.raises(ValueError, match="rate"):
        block_ops._drop_of(1.5)
    with pytest.raises(ValueError, match="rate"):
        block_ops._drop_of(float("nan"))
    with pytest.raises(ValueError, match="rng"):
        block_ops._rng_of(None, 5, x.device)
    with pytest.raises(ValueError, match="int64"):
        block_ops._rng_of(torch.zeros(2), 5, x.device)
    with pytest.raises(ValueError, match="activation"):
        block_ops._act_code("tanh")
    with pytest.raises(ValueError, match="broadcast"):
        block_ops._residual_of(torch.zeros(3), (4, 8), torch.float32)


def test_rate_and_rng_rules():
    assert block_ops._drop_of(0.0) == 0 and block_ops._drop_of(1.0) == 65536 and block_ops._drop_of(0.1) == 6554
    assert block_ops._rng_of((-1, 1 << 65), 5, None)[:2] == ((1 << 64) - 1, 0)
    assert block_ops._rng_of(None, 0, None) == (0, 0, None)


def test_row_views():
    """Leading axes collapse without a copy exactly when one stride serves them."""
    t = torch.arange(2 * 3 * 40.0).view(2, 3, 40)
    m, step = block_ops._rows_of(t[..., 4:20])
    assert step == 40 and m.data_ptr() == t[..., 4:20].data_ptr()
    for view in (t, t[..., 4:20], t.transpose(0, 1), t[:, :2], t[..., ::2], t[:1].expand(4, 3, 40), t[:, :, :1],
                 t.new_zeros(0, 7), torch.arange(5.0), t[0, 0].expand(6, 40)):
        m, step = block_ops._rows_of(view)
        rows = view.reshape(-1, view.shape[-1])
        assert step >= view.shape[-1] and torch.equal(m.as_strided(rows.shape, (step, 1)), rows)


def test_a_forward_mode_tangent_goes_through_autograd():
    """Which has no rule for it and says so; a call past autograd would return no tangent."""
    from torch.autograd import forward_ad
    x, t = torch.zeros(3), torch.ones(3)
    assert not block_ops._records(x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, t)
        assert block_ops._records(None, dual) and block_ops._records(dual)
        assert not block_ops._records(x, None)
        with torch.no_grad():
            assert block_ops._records(x, dual)
    assert block_ops._records(x.clone().requires_grad_())
    with torch.no_grad():
        assert not block_ops._records(x.clone().requires_grad_())


def test_dense_operands_are_aligned():
    """A contiguous view may start anywhere; the kernels' 16-byte accesses may not."""
    from selectssm_b200.ops import _dense
    flat = torch.arange(200.0)
    for t in (flat[3:67].view(2, 4, 8), flat[1:], flat.view(10, 20).t(), flat[4:20].view(4, 4)):
        d = _dense(t)
        assert d.is_contiguous() and d.data_ptr() % 16 == 0 and torch.equal(d, t)
    assert _dense(flat) is flat and _dense(flat[4:20]).data_ptr() == flat[4:20].data_ptr()


def test_a_wait_that_gave_up_is_raised_once(monkeypatch):
    word = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setitem(block_ops._status, 7, (word, ctypes.c_int32.from_address(word.data_ptr())))
    assert block_ops._status_word(7) == word.data_ptr()
    word[0] = _lib.SSM_ERR_TIMEOUT
    with pytest.raises(_lib.SSMLibraryError, match="an earlier dense_act call on cuda:7.*wait"):
        block_ops._status_word(7)
    assert block_ops._status_word(7) == word.data_ptr() and int(word) == 0


def test_dropout_rng_without_the_fused_block_is_refused():
    """The unfused block's dropout draws from torch's generator and would ignore it."""
    from selectssm_b200 import BidirectionalMamba
    m = BidirectionalMamba(32, hidden_features=16, expansion_factor=1, mlp_layer=True)
    with pytest.raises(ValueError, match="fused_block"):
        m(torch.zeros(1, 8, 32), train=True, dropout_rng=(1, 2))


def test_abi_refuses_misaligned_pointers():
    """Which would fault in the kernels' wide accesses."""
    lib = _lib.load()

    def code(f, p):
        return f(ctypes.byref(p), None)

    d = _lib.SSMDenseParams()
    d.rows, d.fin, d.fout = 40, 8, 8
    d.x = d.kernel = d.y = d.dy = d.dx = 0x1000
    for f, query in ((lib.ssm_dense_act_fwd, lib.ssm_dense_fwd_workspace_bytes),
                     (lib.ssm_dense_act_bwd, lib.ssm_dense_bwd_workspace_bytes)):
        d.workspace, d.workspace_bytes = 0x1010, query(ctypes.byref(d)) + 4096
        assert code(f, d) == _lib.SSM_ERR_ALIGN
        d.workspace = None
        for field in ("x", "kernel", "residual", "y", "pre", "dy", "dx", "bias", "dkernel", "dbias", "status"):
            before = getattr(d, field)
            setattr(d, field, 0x1002)
            assert code(f, d) == _lib.SSM_ERR_ALIGN, field
            setattr(d, field, before)
        d.rng = 0x1004
        assert code(f, d) == _lib.SSM_ERR_ALIGN
        d.rng = None
    g = _lib.SSMGroupNormParams()
    g.batch, g.seqlen, g.dim, g.groups = 2, 5, 33, 3
    g.x = g.y = g.dy = g.dx = g.stats = 0x1000
    for f, query in ((lib.ssm_group_norm_act_fwd, lib.ssm_group_norm_fwd_workspace_bytes),
                     (lib.ssm_group_norm_act_bwd, lib.ssm_group_norm_bwd_workspace_bytes)):
        g.workspace, g.workspace_bytes = 0x1010, query(ctypes.byref(g)) + 4096
        assert code(f, g) == _lib.SSM_ERR_ALIGN
        g.workspace = None
        for field, bad in (("x", 0x1002), ("y", 0x1002), ("dy", 0x1002), ("dx", 0x1002), ("scale", 0x1002),
                           ("bias", 0x1002), ("stats", 0x1004), ("dscale", 0x1002), ("dbias", 0x1002)):
            before = getattr(g, field)
            setattr(g, field, bad)
            assert code(f, g) == _lib.SSM_ERR_ALIGN, field
            setattr(g, field, before)
    p = _lib.SSMDropoutParams()
    p.rows, p.dim = 2, 8
    p.x = p.y = p.dy = p.dx = 0x1000
    for f in (lib.ssm_dropout_act_fwd, lib.ssm_dropout_act_bwd):
        for field, bad in (("x", 0x1002), ("residual", 0x1002), ("y", 0x1002), ("dy", 0x1002), ("dx", 0x1002), ("rng", 0x1004)):
            before = getattr(p, field)
            setattr(p, field, bad)
            assert code(f, p) == _lib.SSM_ERR_ALIGN, field
            setattr(p, field, before)
