"""The C entries of the answer path refuse what they cannot do before anything is enqueued (no GPU needed), and the Python
entries refuse CPU tensors."""
import pytest
import torch

from generative_recommenders_amd import enc_ops, hmx, mx_ops

P = 0x1000                  # a 16-byte aligned non-null address that a refused call never reads
EINVAL = -1


def test_norm_entries():
    L = hmx.lib()
    good = dict(x=P, ldx=64, r=P, ldr=64, w=P, T=4, d=64, eps=1e-6, bf16=0)
    for bad in (dict(x=None), dict(w=None), dict(T=-1), dict(d=0), dict(d=32769), dict(eps=-1.0), dict(eps=float("nan")),
                dict(ldx=-1), dict(ldr=-1)):
        a = list({**good, **bad}.values())
        assert L.hmx_add_rmsnorm_fwd(*a, P, P, None, None) == EINVAL
        assert L.hmx_add_rmsnorm_mx8(*a, P, P, P, None) == EINVAL
    a = list(good.values())
    assert L.hmx_add_rmsnorm_fwd(*a, None, P, None, None) == EINVAL          # a residual without a place for the sum
    assert L.hmx_add_rmsnorm_fwd(*a, P, None, None, None) == EINVAL
    assert L.hmx_add_rmsnorm_mx8(*a, P, None, P, None) == EINVAL
    bwd = dict(s=P, w=P, rstd=P, dy=P, ds=None, T=4, d=64, bf16=0, dx=P, dw=None, ws=None, ws_bytes=0, stream=None)
    for bad in (dict(s=None), dict(w=None), dict(rstd=None), dict(dy=None), dict(dx=None), dict(T=-1), dict(d=40000)):
        assert L.hmx_add_rmsnorm_bwd(*{**bwd, **bad}.values()) == EINVAL
    nbytes = L.hmx_add_rmsnorm_bwd_workspace_bytes(10 ** 5, 64)
    assert nbytes > 0 and L.hmx_add_rmsnorm_bwd_workspace_bytes(4, 64) == 0
    for bad in (dict(dw=P), dict(dw=P, ws=P, ws_bytes=nbytes - 1), dict(dw=P, ws=None, ws_bytes=nbytes)):
        assert L.hmx_add_rmsnorm_bwd(*{**bwd, "T": 10 ** 5, **bad}.values()) == -2
    assert L.hmx_add_rmsnorm_fwd(None, 64, None, 0, None, 0, 64, 0.0, 0, None, None, None, None) == 0
    assert L.hmx_add_rmsnorm_bwd(*{**bwd, "T": 0, "s": None}.values()) == 0


def test_mx4_entries():
    L = hmx.lib()
    assert L.hmx_mx4_quantize(P, 64, -1, 64, 0, P, P, None) == EINVAL
    assert L.hmx_mx4_quantize(P, 64, 4, 0, 0, P, P, None) == EINVAL
    assert L.hmx_mx4_quantize(P, 64, 4, 64, 0, P + 4, P, None) == EINVAL     # codes not aligned
    assert L.hmx_mx4_quantize(None, 64, 4, 64, 0, P, P, None) == EINVAL
    assert L.hmx_mx4_quantize(None, 64, 0, 64, 0, None, None, None) == 0
    assert L.hmx_mx_dequantize(P, P, 4, 64, 6, 0, P, None) == EINVAL
    assert L.hmx_mx_dequantize(P, None, 4, 64, 4, 0, P, None) == EINVAL
    good = dict(x=P, ldx=64, xs=None, kind=0, M=4, codes=P, scales=P, N=8, K=64, bf16=0, out=P, ws=None, ws_bytes=0, stream=None)
    for bad in (dict(x=None), dict(kind=3), dict(kind=2), dict(xs=P), dict(kind=2, xs=P, K=60), dict(M=-1), dict(N=-1), dict(K=0),
                dict(codes=P + 8), dict(scales=None), dict(out=None), dict(N=1 << 40), dict(M=1 << 30), dict(ldx=-1)):
        assert L.hmx_linear_mx4(*{**good, **bad}.values()) == EINVAL, bad
    nbytes = L.hmx_linear_mx4_workspace_bytes(0, 4, 1000)
    assert nbytes > 0 and L.hmx_linear_mx4_workspace_bytes(0, 4, 128) == 0
    for bad in (dict(ws=P, ws_bytes=nbytes - 1), dict(ws=None, ws_bytes=nbytes), dict(ws=P + 8, ws_bytes=nbytes)):
        assert L.hmx_linear_mx4(*{**good, "K": 1000, "ldx": 1000, **bad}.values()) == -2
    assert L.hmx_linear_mx4(*{**good, "M": 0}.values()) == 0


def test_python_entries_refuse_cpu_tensors():
    x, w = torch.zeros(4, 64), torch.ones(64)
    for call in (lambda: enc_ops.add_rmsnorm(x, x, w), lambda: mx_ops.add_rmsnorm_mx8(x, x, w), lambda: mx_ops.quantize_mx4(x),
                 lambda: mx_ops.dequantize_mx4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)),
                 lambda: mx_ops.linear_mx4(x, torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8))):
        with pytest.raises(hmx.HmxError):
            call()


def test_sample_entry():
    L = hmx.lib()
    good = dict(logits=P, ld=64, B=4, V=64, bf16=0, u=P, u64=0, draws=1, t=None, k=None, p=None, mp=None, ta=1.0, ka=0, pa=1.0,
                mpa=0.0, ids=P, probs=P, ws=None, ws_bytes=0, stream=None)
    for bad in (dict(logits=None), dict(ld=-1), dict(B=-1), dict(V=0), dict(V=1 << 31), dict(u=None), dict(draws=-1),
                dict(ids=None), dict(probs=None), dict(B=1 << 22)):
        assert L.hmx_sample_logits(*{**good, **bad}.values()) == EINVAL, bad
    nbytes = L.hmx_sample_logits_workspace_bytes(4, 1 << 20)
    assert nbytes > 0 and L.hmx_sample_logits_workspace_bytes(4, 64) == 0
    for bad in (dict(ws=P, ws_bytes=nbytes - 1), dict(ws=None, ws_bytes=nbytes), dict(ws=P + 8, ws_bytes=nbytes)):
        assert L.hmx_sample_logits(*{**good, "V": 1 << 20, "ld": 1 << 20, **bad}.values()) == -2
    assert L.hmx_sample_logits(*{**good, "B": 0, "logits": None}.values()) == 0
    assert L.hmx_sample_logits(*{**good, "draws": 0}.values()) == 0
