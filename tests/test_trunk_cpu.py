"""Refusals of the residual-trunk operators: decided on the host, before any launch, hence testable without a GPU."""
import ctypes as C

import pytest
import torch

from scpair_amd import _lib, ops

X, H = torch.zeros(4, 8), torch.zeros(4, 8)


@pytest.mark.parametrize("args,kw", [
    ((torch.zeros(()),), {}),
    ((X.half(),), {}),
    ((X.double(), H.double()), {}),
    ((X.bfloat16(), H), {}),                                         # a bf16 stream needs bf16 blocks
    ((X, torch.zeros(4, 7)), {}),
    ((X, torch.zeros(1, 8)), {}),
    ((X, H), {"pre": None}),
    ((X, H), {"pre": "batch"}),
    ((X, H), {"post": "batch"}),
    ((X, H), {"gate_act": "relu"}),
    ((X, H), {"eps": 0.0}),
    ((X, H), {"eps": float("nan")}),
    ((X, H), {"out_dtype": torch.bfloat16}),
    ((X, H), {"pre": "rms", "pre_bias": torch.zeros(8)}),
    ((X, H), {"post": "rms", "post_bias": torch.zeros(8)}),
    ((X, H), {"post_weight": torch.ones(8)}),
    ((X, H), {"pre_weight": torch.ones(7)}),
    ((X, H), {"pre_weight": torch.ones(8, dtype=torch.int32)}),
    ((X, H), {"scale": torch.ones(7)}),
    ((X, H), {"gate": torch.zeros(4)}),
    ((X, H), {"gate": torch.zeros(3, 8)}),
    ((X, H), {"gate": torch.zeros(4, 8, dtype=torch.bfloat16)}),     # a full gate has h's type
    ((X,), {"gate": X}),
    ((X,), {"scale": 0.5}),
    ((X,), {"post": "rms"}),
    ((X.bfloat16(),), {"out_dtype": torch.float32}),
    ((torch.zeros(2, 0), torch.zeros(2, 0)), {}),
    ((torch.zeros(1, 16385),), {}),
])
def test_gated_residual_norm_refuses(args, kw):
    with pytest.raises(ValueError):
        ops.gated_residual_norm(*args, **kw)


def test_gated_residual_norm_has_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.gated_residual_norm(X, H)


def test_residual_norm_c_entry_refuses():
    L = _lib.lib()
    assert L.scp_residual_norm_max_cols() == 16384

    def args(**kw):
        a = _lib.ResidualNorm()
        base = dict(x=64, h=64, r=64, y=64, stats=64, rows=2, cols=8, pre=1, ldx=8, ldh=8, eps=1e-5)
        for k, v in (base | kw).items():
            setattr(a, k, v)
        return C.byref(a)

    assert L.scp_residual_norm_fwd(None, None) == -1
    for bad in (dict(rows=0), dict(cols=0), dict(x=None), dict(ldx=-1), dict(pre=0), dict(pre=3), dict(post=3), dict(x_bf16=1),
                dict(gate_mode=4, gate=64), dict(gate_mode=1), dict(gate_act=3), dict(scale_mode=1), dict(y=None), dict(r=None),
                dict(h=None, post=1)):
        assert L.scp_residual_norm_fwd(args(**bad), None) == -1, bad
        assert L.scp_last_error()
    assert L.scp_residual_norm_fwd(args(cols=16385), None) == -2
    for bad in (dict(stats=None), dict(dw2=64), dict(dw1=64, ws=64), dict(dscale=64, ws=64), dict(dgate=64),
                dict(dy=64, lddy=-8)):
        assert L.scp_residual_norm_bwd(args(**bad), None) == -1, bad
    assert L.scp_residual_norm_bwd_ws_floats(0, 8) == 0
    assert L.scp_residual_norm_bwd_ws_floats(1, 900) == 5 * 900


@pytest.mark.parametrize("call", [
    lambda: ops.pack8(torch.zeros(())),
    lambda: ops.pack8(torch.zeros(3, 4, dtype=torch.float16)),
    lambda: ops.pack8(3.0),
    lambda: ops.unpack8(torch.zeros(3)),
    lambda: ops.unpack8(ops.Packed8(torch.zeros(1, 64, dtype=torch.int8), torch.zeros(1, 1, dtype=torch.uint8), (1, 64),
                                    torch.float32), torch.float64),
    lambda: ops.unpack8(ops.Packed8(torch.zeros(1, 64, dtype=torch.int8), torch.zeros(1, 1, dtype=torch.uint8), (2, 64),
                                    torch.float32)),
    lambda: ops.unpack8(ops.Packed8(torch.zeros(1, 128, dtype=torch.int8)[:, ::2], torch.zeros(1, 1, dtype=torch.uint8), (1, 64),
                                    torch.float32)),
    lambda: ops.unpack8(ops.Packed8(torch.zeros(1, 64, dtype=torch.int8), torch.zeros(1, 2, dtype=torch.uint8), (1, 64),
                                    torch.float32)),
    lambda: ops.act8(torch.zeros(3, 4, dtype=torch.float64)),
    lambda: ops.act8(torch.zeros(3, 4), "tanh"),
    lambda: ops.linear8(torch.zeros(3, 4), torch.zeros(5, 3)),
    lambda: ops.linear8(torch.zeros(3, 4), torch.zeros(4)),
    lambda: ops.linear8(torch.zeros(3, 0), torch.zeros(5, 0)),
    lambda: ops.linear8(torch.zeros(3, 4), torch.zeros(0, 4)),
    lambda: ops.linear8(torch.zeros(3, 4), torch.zeros(5, 4, dtype=torch.bfloat16)),
    lambda: ops.linear8(torch.zeros(3, 4, dtype=torch.float16), torch.zeros(5, 4)),
    lambda: ops.linear8(torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(4)),
    lambda: ops.linear8(torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(5, dtype=torch.int64)),
    lambda: ops.linear8(torch.zeros(1, 32768), torch.zeros(1).expand(32768, 32768)),
])
def test_checkpoint_operators_refuse(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("call", [lambda: ops.pack8(X), lambda: ops.act8(X), lambda: ops.linear8(X, torch.zeros(5, 8))])
def test_checkpoint_operators_have_no_cpu_path(call):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()


def test_checkpoint_c_entries_refuse():
    L = _lib.lib()
    a = 4096
    assert L.scp_pack8(None, 0, 8, 2, 8, a, a, None) == -1 and L.scp_pack8(a, 0, 8, 0, 8, a, a, None) == -1
    assert L.scp_pack8(a, 0, 8, 2, 8, a + 1, a, None) == -1 and L.scp_pack8(a, 0, -8, 2, 8, a, a, None) == -1
    assert L.scp_pack8(a, 0, 8, 2, (1 << 24) + 1, a, a, None) == -2
    assert L.scp_unpack8(a, None, 2, 8, a, 0, None) == -1 and L.scp_unpack8(a, a, 2, 8, None, 0, None) == -1
    assert L.scp_act8_fwd(a, 0, 8, 2, 8, 3, 0.0, a, a, a, None) == -1 and L.scp_act8_fwd(a, 0, 8, 2, 8, 0, 0.0, a, a, None, None) == -1
    assert L.scp_act8_bwd(a, a, 2, 8, -1, 0.0, a, 0, 8, a, None) == -1 and L.scp_act8_bwd(a, a, 2, 8, 0, 0.0, None, 0, 8, a, None) == -1
    assert L.scp_gemm_rows(2, 8, 8, 8, a, 8, a, 8, a, 1, 8, None, None, None) == -1
    assert L.scp_gemm_rows(0, 8, 8, 9, a, 8, a, 16, a, 1, 8, None, None, None) == -1
    assert L.scp_gemm_rows(0, 8, 8, 8, a + 2, 8, a, 8, a, 0, 8, None, None, None) == -1
    assert L.scp_gemm_rows(0, 1 << 20, 8, 1024, a, 1024, a, 1024, a, 1, 8, None, None, None) == -2
    assert L.scp_gemm_q8(8, 8, 8, a, 8, a, None, a, 0, 8, None, None) == -1
    assert L.scp_gemm_q8(9, 8, 8, a, 8, a, a, a, 0, 8, None, None) == -1
    assert L.scp_gemm_q8(8, 8, 8, a, 12, a, a, a, 0, 8, None, None) == -1
    assert L.scp_gemm_q8(8, 8, 8, a, 8, a, a, a, 0, 7, None, None) == -1
    # a batch of 4 M rows needs K-ranges below 2 GiB, hence slabs
    assert L.scp_gemm_q8_ws_floats(1024, 1024, 4_000_000, 1024, 1024) >= 8 * 1024 * 1024
    assert L.scp_gemm_q8(1024, 1024, 4_000_000, a, 1024, a, a, a, 0, 1024, None, None) == -1
    assert b"workspace" in L.scp_last_error()


def test_linear8_c_entries_refuse():
    L = _lib.lib()

    def args(**kw):
        a = _lib.Linear8()
        for k, v in (dict(x=4096, W=4096, y=4096, dy=4096, M=5, N=8, K=16, ldx=16, lddy=8, ns=3, ws=4096) | kw).items():
            setattr(a, k, v)
        return C.byref(a)

    for bad in (dict(M=0), dict(N=0), dict(K=0), dict(w_bf16=1), dict(ns=2), dict(codes=4096), dict(codes=4097, steps=4096)):
        assert L.scp_linear8_fwd(args(**bad), None) == -1 and L.scp_linear8_bwd(args(**bad), None) == -1, bad
        assert L.scp_linear8_fwd_ws(args(**bad)) == -1 and L.scp_linear8_bwd_ws(args(**bad)) == -1, bad
    for bad in (dict(M=1 << 30), dict(K=(1 << 20) + 1), dict(N=40000, K=40000)):
        assert L.scp_linear8_fwd(args(**bad), None) == -2 and L.scp_linear8_fwd_ws(args(**bad)) == -1, bad
    split = dict(M=64, N=4096, K=4096, ldx=4096, lddy=4096)          # few tiles, long sums: K-ranges, hence slabs
    assert L.scp_linear8_fwd_ws(args(**split)) > 0 and L.scp_linear8_bwd_ws(args(**split, dx=4096)) > 0
    for bad in (dict(x=None), dict(W=None), dict(y=None), dict(ldx=-1), dict(split, ws=None), dict(split, ws=4096 + 16)):
        assert L.scp_linear8_fwd(args(**bad), None) == -1, bad
    for bad in (dict(dy=None), dict(lddy=-1), dict(dx=4096, W=None), dict(dW=4096), dict(split, dx=4096, ws=None),
                dict(db=4096, ws=None)):
        assert L.scp_linear8_bwd(args(**bad), None) == -1, bad
    # aligned bf16 operands need no copies, and a large product no slabs
    big = dict(x_bf16=1, w_bf16=1, M=16384, N=4096, K=4096, ldx=4096, lddy=4096, dx=4096, dW=4096, codes=4096, steps=4096)
    assert L.scp_linear8_fwd_ws(args(**big)) == 0 and L.scp_linear8_bwd_ws(args(**big)) == 0

    # rows too far apart for a tile's 32-bit offsets are copied, whatever the tile
    for far in (1 << 25, 1 << 30, 1 << 33):
        rows = dict(x_bf16=1, w_bf16=1, M=4096, N=4096, K=4096, lddy=4096)
        assert L.scp_linear8_fwd_ws(args(**rows, ldx=far)) >= 4096 * 4096 * 2 > L.scp_linear8_fwd_ws(args(**rows, ldx=4104))


@pytest.mark.parametrize("args,kw", [((0, 1), {}), ((16385, 1), {}), ((8, 0), {}), ((8, 1), {"norm": "batch"}),
                                     ((8, 1), {"gate": "none"}), ((8, 1), {"activation": "relu6"}),
                                     ((8, 1), {"block_dtype": torch.float16})])
def test_residual_trunk_refuses(args, kw):
    import scpair_amd as S
    with pytest.raises(ValueError):
        S.ResidualTrunk(*args, **kw)


def test_residual_trunk_parameters():
    import scpair_amd as S
    names = {n for n, _ in S.ResidualTrunk(8, 2, gate="sigmoid").named_parameters()}
    assert {"fc1.1.weight", "fc2.0.bias", "pre_weight.2", "pre_bias.2", "post_weight.1", "post_bias.1", "scale.1", "gate.1"} <= names
    names = {n for n, _ in S.ResidualTrunk(8, 1, norm="rms").named_parameters()}
    assert not any("norm" in n or "_bias" in n or "gate" in n for n in names)
