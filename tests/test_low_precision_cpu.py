"""Refusals of the low-precision and router-loss entry points that need no GPU, and the host-side weight preparation."""
import ctypes

import pytest
import torch

_BUF = ctypes.create_string_buffer(4096)
P = (ctypes.addressof(_BUF) + 255) // 256 * 256  # aligned; never dereferenced: every call below is rejected first


def _lib():
    from layered_prefill_b200 import _lib
    return _lib.lib, _lib.last_error


def test_norm_quant_refusals():
    lib, err = _lib()
    f = lib.moe_b200_rms_norm_quant_fp8
    assert f(P, P, None, None, None, P, P, 1e-6, 0, 256, 128, None) == 0  # no token
    for args in ((4, 100, -1), (4, 0, -1), (-1, 256, 128), (4, 32776, -1), (4, 256, 64), (4, 264, 128), (4, 256, 0)):
        assert f(P, P, None, None, None, P, P, 1e-6, *args, None) == 1, args
    assert f(P, P, None, None, P, P, P, 1e-6, 4, 256, 128, None) == 1 and "null" in err()  # a residual without its output
    assert f(None, P, None, None, None, P, P, 1e-6, 4, 256, 128, None) == 1
    for i in (0, 2, 5, 6):
        ptrs = [P, P, P, None, None, P, P]
        ptrs[i] += 2
        assert f(*ptrs, 1e-6, 4, 256, 128, None) == 1 and "16 bytes" in err()
    assert f(P, P, None, P + 8, P, P, P, 1e-6, 4, 256, 128, None) == 1


def test_w4_linear_refusals():
    lib, err = _lib()
    room = lib.moe_b200_w4_linear_workspace_bytes

    def f(out, x, ld, q, s, z, b, M, N, K, g, stream, ws=P, ws_bytes=1 << 30):
        return lib.moe_b200_w4_linear(out, x, ld, q, s, z, b, M, N, K, g, ws, ws_bytes, stream)

    assert f(P, P, 256, P, P, None, None, 0, 8, 256, 64, None) == 0
    for ld, (M, N, K, g) in ((256, (1, 8, 256, 48)), (256, (1, 8, 224, 64)), (256, (-1, 8, 256, 64)), (256, (1, 0, 256, 64)),
                             (260, (2, 8, 256, 64)), (0, (2, 8, 256, 64)), (128, (2, 8, 256, 64)), (256, (1, 8, 0, 64))):
        assert f(P, P, ld, P, P, None, None, M, N, K, g, None) == 1, (ld, M, N, K, g)
    assert f(P, P + 2, 256, P, P, None, None, 1, 8, 256, 64, None) == 1 and "16 bytes" in err()
    assert f(P, P, 256, P + 8, P, None, None, 1, 8, 256, 64, None) == 1
    assert f(P, P, 256, P, None, None, None, 1, 8, 256, 64, None) == 1 and "null" in err()
    assert f(P, P, 256, P, P, None, None, 1 << 30, 8, 256, 64, None) == 1 and "sizes" in err()
    need = room(16, 8192, 64)
    assert need > 16 * 8192 * 2 and room(1, 2048, 128) == 0 and room(0, 2048, 128) == 0 and room(64, 8192, 48) == 0
    assert f(P, P, 8192, P, P, None, None, 16, 8, 8192, 64, None, P, need - 1) == 3 and "workspace" in err()
    assert f(P, P, 8192, P, P, None, None, 16, 8, 8192, 64, None, P + 8, need) == 3


def test_w4_experts_refusals():
    lib, err = _lib()
    f, need = lib.moe_b200_fused_experts_w4, lib.moe_b200_fused_experts_w4_workspace_bytes(4, 8, 2, 256, 128)
    assert need > 0 and lib.moe_b200_fused_experts_w4_workspace_bytes(4, 0, 2, 256, 128) == 0

    def call(x=P, z13=None, z2=None, T=4, E=8, k=2, H=256, I=128, g=64, act=0, ws=P, ws_bytes=need, out=P):
        return f(x, P, P, z13, None, P, P, z2, None, P, P, out, T, E, k, H, I, g, act, ws, ws_bytes, None)

    assert call(T=0) == 0
    for bad in (dict(g=16), dict(H=240), dict(I=96), dict(act=2), dict(k=9), dict(x=None), dict(out=None), dict(z13=P), dict(z2=P),
                dict(x=P + 2), dict(T=-1)):
        assert call(**bad) == 1, bad
    assert call(ws_bytes=need - 1) == 3 and call(ws=None) == 3 and "workspace" in err()
    assert lib.moe_b200_fused_experts_fp8_quantized(P, None, P, P, P, P, P, P, P, 4, 8, 2, 256, 128, 0, 128, P, 1 << 30, P, None) == 1


def test_router_refusals():
    lib, err = _lib()
    f, b = lib.moe_b200_router_loss, lib.moe_b200_router_backward
    need = lib.moe_b200_router_loss_workspace_bytes(640, 16)
    assert need > 0 and lib.moe_b200_router_loss_workspace_bytes(128, 16) == 0
    assert f(P, P, P, P, P, 0, P, None, 64, 16, 17, P, need, None) == 1
    assert f(P, P, P, P, P, 0, P, None, 64, 1025, 2, P, 1 << 30, None) == 1 and "experts" in err()
    assert f(P, P, P, P, None, 0, P, None, 64, 16, 2, P, need, None) == 1
    assert f(P, P, P, P, P, 0, P, None, 640, 16, 2, P, need - 1, None) == 3
    assert b(P, P, 0, P, P, P, P, P, None, 0, 16, 2, 1, None) == 0
    assert b(P, P, 0, P, None, P, P, P, None, 4, 16, 2, 1, None) == 1
    assert b(P, P, 0, None, P, P, P, P, None, 4, 16, 2, 1, None) == 1
    assert b(P, P, 0, P, P, P, P, P, None, 4, 16, 0, 1, None) == 1


def test_cpu_tensors_are_refused():
    from layered_prefill_b200 import fused_moe, ops
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.rms_norm_quant_fp8(torch.zeros(2, 256, dtype=torch.float8_e4m3fn), torch.zeros(2, 2), x, x[0], 1e-6)
    q, s, _ = fused_moe.quant_w4(torch.randn(8, 256), 64)
    with pytest.raises(RuntimeError):
        ops.w4_linear(torch.zeros(2, 8, dtype=torch.bfloat16), x, q, s)
    with pytest.raises(RuntimeError):
        fused_moe.fused_topk_with_loss(torch.zeros(2, 4), 2, True)


def test_more_tokens_than_an_int_counts_are_refused():
    """2^32 + 1 would cross the C interface as 1. The tensors are one row seen many times."""
    from layered_prefill_b200 import ops
    T = 2**32 + 1
    row = lambda n, dtype: torch.zeros(1, n, dtype=dtype).expand(T, n)  # noqa: E731
    bf16 = torch.bfloat16
    with pytest.raises(RuntimeError, match="at most"):
        ops.rms_norm_quant_fp8(row(8, torch.float8_e4m3fn), row(1, torch.float32), row(8, bf16), torch.zeros(8, dtype=bf16), 1e-6, -1)
    with pytest.raises(RuntimeError, match="at most"):
        ops.w4_linear(row(8, bf16), row(32, bf16), torch.zeros(8, 16, dtype=torch.uint8), torch.zeros(8, 1, dtype=bf16))
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="at most"):
        ops.router_loss(torch.zeros(2), one, one, torch.zeros(1), row(1, torch.float32), row(1, torch.int32))
    with pytest.raises(RuntimeError, match="at most"):
        ops.router_backward(row(1, torch.float32), row(1, torch.float32), row(1, torch.int32), one, one, None, None, True)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zero_points", [False, True])
def test_quant_w4_is_within_half_a_step(group, zero_points):
    from layered_prefill_b200 import fused_moe
    g = torch.Generator().manual_seed(group)
    w = torch.randn(3, 20, 256, generator=g) * 0.05 + 0.02
    w[0, 0] = 0
    codes, scale, zero = fused_moe.quant_w4(w, group, zero_points)
    assert codes.shape == (3, 20, 128) and codes.dtype == torch.uint8 and scale.dtype == torch.bfloat16
    assert (zero is None) == (not zero_points)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    s = scale.float().repeat_interleave(group, -1)
    back = (code - (8.0 if zero is None else zero.float().repeat_interleave(group, -1))) * s
    # half a step inside the range; at its ends the bf16 scale (2^-8) and the zero point's own half step move it by up to 15 * 2^-8
    # and half a step more, and the positive end of the symmetric range (code 15 = 7 steps of 7.5) by half a step
    assert ((back - w).abs() <= (1.0 + 16 * 2.0 ** -8) * s + 1e-12).all()
    assert (back - w).norm() / w.norm() < 0.15
    assert (back[0, 0] == 0).all()
    with pytest.raises(ValueError):
        fused_moe.quant_w4(w, 48)


def test_expert_shards_put_together_are_the_whole():
    from layered_prefill_b200 import fused_moe
    E, I, H, g = 4, 256, 128, 64
    gen = torch.Generator().manual_seed(1)
    w13, w2 = (fused_moe.quant_w4(torch.randn(*s, generator=gen), g, True) for s in ((E, 2 * I, H), (E, H, I)))
    parts = [fused_moe.shard_w4_expert_weights(w13, w2, r, 4, g) for r in range(4)]
    for i in range(3):
        assert torch.equal(torch.cat([p[0][i][:, :I // 4] for p in parts] + [p[0][i][:, I // 4:] for p in parts], 1), w13[i])
        assert torch.equal(torch.cat([p[1][i] for p in parts], 2), w2[i])
    with pytest.raises(ValueError):
        fused_moe.shard_w4_expert_weights(w13, w2, 0, 8, g)  # shares of 32 columns, groups of 64


def test_w4_row_parallel_linear_loads_and_refuses():
    from layered_prefill_b200 import fused_moe, linear
    layer = linear.W4RowParallelLinear(256, 24, bias=True, group_size=64)
    assert layer.zeros is None and not hasattr(layer, "weight")
    q, s, _ = fused_moe.quant_w4(torch.randn(24, 256), 64)
    layer.qweight.weight_loader(layer.qweight, q)
    layer.scales.weight_loader(layer.scales, s)
    layer.bias.weight_loader(layer.bias, torch.ones(24))
    assert torch.equal(layer.qweight, q) and torch.equal(layer.scales, s) and (layer.bias == 1).all()
    layer.tp_rank, layer.tp_size = 1, 2  # the second rank's columns of a layer twice as wide
    q2, s2, _ = fused_moe.quant_w4(torch.randn(24, 512), 64)
    layer.qweight.weight_loader(layer.qweight, q2)
    layer.scales.weight_loader(layer.scales, s2)
    assert torch.equal(layer.qweight, q2[:, 128:]) and torch.equal(layer.scales, s2[:, 4:])
    with pytest.raises(ValueError):
        linear.W4RowParallelLinear(192, 8, group_size=128)


@pytest.mark.parametrize("activation", ["silu", "swigluoai"])
@pytest.mark.parametrize("tp", [2, 4])
def test_expert_shards_add_up_to_the_whole(activation, tp):
    """The partial results of the ranks, each from its own shard, sum to the unsharded experts' result."""
    from layered_prefill_b200 import fused_moe
    E, I, H, g = 3, 128, 64, 32
    gen = torch.Generator().manual_seed(tp)
    w13, w2 = (fused_moe.quant_w4(torch.randn(*s, generator=gen) * 0.2, g, True) for s in ((E, 2 * I, H), (E, H, I)))
    x = torch.randn(5, H, generator=gen, dtype=torch.float64)

    def dense(w):
        codes, scale, zero = w
        code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
        return (code - zero.double().repeat_interleave(g, -1)) * scale.double().repeat_interleave(g, -1)

    def experts(a, b):  # [E, T, H]: every token through every expert
        gu = torch.einsum("th,enh->etn", x, dense(a))
        if activation == "silu":
            gate, up = gu.chunk(2, -1)
            h = gate * torch.sigmoid(gate) * up
        else:  # gate and up rows alternate
            gate, up = gu[..., 0::2].clamp(max=7), gu[..., 1::2].clamp(-7, 7)
            h = gate * torch.sigmoid(1.702 * gate) * (up + 1)
        return torch.einsum("eti,ehi->eth", h, dense(b))

    whole = experts(w13, w2)
    parts = [fused_moe.shard_w4_expert_weights(w13, w2, r, tp, g, activation) for r in range(tp)]
    assert all(t.is_contiguous() for p in parts for triple in p for t in triple)
    # 64-bit sums of I + H terms in another order
    assert (sum(experts(*p) for p in parts) - whole).abs().max() <= (I + H) * 2.0 ** -52 * whole.abs().max() * 16
    with pytest.raises(ValueError):
        fused_moe.shard_w4_expert_weights(w13, w2, 0, tp, g, "gelu")


def test_w4_row_parallel_linear_has_a_bf16_bias_and_no_dense_weight(monkeypatch):
    from layered_prefill_b200 import linear
    assert torch.get_default_dtype() == torch.float32
    sizes, empty = [], torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: sizes.append(empty(*a, **k).nbytes) or empty(*a, **k))
    layer = linear.W4RowParallelLinear(256, 24, bias=True, group_size=64, zero_points=True)
    assert layer.bias.dtype == torch.bfloat16 and not layer.bias.requires_grad and not hasattr(layer, "weight")
    assert max(sizes) == 24 * 128  # the codes
    assert [n for n, _ in layer.named_parameters()] == ["qweight", "scales", "zeros", "bias"]
    assert all(callable(p.weight_loader) for p in layer.parameters())
    assert linear.W4RowParallelLinear(256, 24, group_size=64).bias is None
    dense = linear.RowParallelLinear(256, 24, bias=True)  # as it was: both in the default type
    assert dense.weight.shape == (24, 256) and dense.weight.dtype == dense.bias.dtype == torch.float32


def test_outputs_over_inputs_are_refused():
    """Inputs are read while outputs are written: a result over its input would depend on which block comes first."""
    lib, err = _lib()
    far = P + (1 << 20)  # never dereferenced either

    def linear(out, x, M, ld, N=128, K=128):
        return lib.moe_b200_w4_linear(out, x, ld, P, P, None, None, M, N, K, 64, None, 0, None)

    for out, x, M, ld in ((far, far, 1, 128), (far, far, 4, 128), (far + 3 * 256, far, 4, 128), (far, far + 4 * 256 - 16, 4, 128),
                          (far + 256, far, 2, 512)):
        assert linear(out, x, M, ld) == 1 and "overlap" in err(), (out - far, x - far, M, ld)
    for x, grad, bf16 in ((far, far, 0), (far + 4 * 64 - 4, far, 0), (far, far + 4 * 32 - 2, 1)):
        assert lib.moe_b200_router_backward(grad, x, bf16, P, P, P, P, P, None, 4, 16, 2, 1, None) == 1 and "overlap" in err()
    need = lib.moe_b200_fused_experts_w4_workspace_bytes(4, 8, 2, 256, 128)
    for out in (far + 512, far - 512, far + 8):
        assert lib.moe_b200_fused_experts_w4(far, P, P, None, None, P, P, None, None, P, P, out, 4, 8, 2, 256, 128, 64, 0, P, need,
                                             None) == 1 and "overlap" in err()


def test_where_the_library_asks_for_no_workspace():
    """ops.py does not ask the library below these sizes: nothing may be needed there, and the losses' rule is exact."""
    from layered_prefill_b200 import ops
    lib, _ = _lib()
    for T in (0, 1, 2, 63, 127, 128, 129, 200, 5000):
        for E in (1, 8, 100, 127, 128, 129, 160, 256, 1023, 1024):
            room = lib.moe_b200_router_loss_workspace_bytes(T, E) > 0
            assert room == (T > ops._LOSS_ALONE_TOKENS or T * E > ops._LOSS_ALONE_LOGITS), (T, E)
    for group in (32, 64, 128):
        for K in (group, 128, 256, 384, 1024, 2048, 4096, 7936, 8064, 8192, 16384):
            for M in range(1, 66):
                if M * (K + 127) <= ops._W4_SMALL:
                    assert lib.moe_b200_w4_linear_workspace_bytes(M, K, group) == 0, (M, K, group)
