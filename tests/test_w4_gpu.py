"""Products with 4-bit weights and group scales, dense and over the routed experts, against the same products in 64 bits.

Tolerances. A sum of K products in fp32, in any order and with a truncating adder, is off by at most (K / 16 + 64) * 2^-23 of
sum |w x|: products of a tensor instruction are exact and added 16 at a time, and at most 64 further additions (groups, warps) follow.
The output's rounding adds 2^-8 of the value.
Activations become 16-bit integers times 2^(e - 14), 2^e being the power of two at or below the largest |x| of 128 columns: a step of
at most 2^-14 of the largest, so half a step is at most 2^-15 of it, which adds 2^-15 * largest * sum |w|. A bf16 value of exponent at
least e - 7 is a whole number of steps (its last bit is worth 2^(e - 7 - 7)) and adds nothing: only values below 2^-7 * 2^e, which are
below 2^-7 of the largest, do. The experts' intermediate is fp32 and adds it everywhere."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8


def _gamma(K):
    return (K / 16 + 64) * 2.0 ** -23


def _weights(N, K, group, zeros, g, lead=()):
    packed = torch.randint(0, 256, (*lead, N, K // 2), generator=g, dtype=torch.uint8)
    scale = (0.01 * torch.exp(0.5 * torch.randn(*lead, N, K // group, generator=g))).to(torch.bfloat16)
    zp = torch.randint(0, 16, (*lead, N, K // group), generator=g, dtype=torch.uint8) if zeros else None
    return packed.cuda(), scale.cuda(), None if zp is None else zp.cuda()


def _dense64(packed, scale, zp, group):
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).double()
    z = 8.0 if zp is None else zp.double().repeat_interleave(group, -1)
    return (code - z) * scale.double().repeat_interleave(group, -1)


def _step(x):
    """2^-15 of the largest |x| of every 128 columns, [.., K]."""
    pad = -x.size(-1) % 128
    big = torch.nn.functional.pad(x.abs(), (0, pad)).unflatten(-1, (-1, 128)).amax(-1)
    return 2.0 ** -15 * big.repeat_interleave(128, -1)[..., :x.size(-1)]


def _bf16_off(x):
    """What a bf16 x may be off by as an integer."""
    return torch.where(x.abs() < 2.0 ** 8 * _step(x), _step(x), torch.zeros_like(x))


def _linear(x, packed, scale, zp, bias=None):
    from layered_prefill_b200 import ops
    out = torch.full((*x.shape[:-1], packed.size(0)), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.w4_linear(out, x, packed, scale, zp, bias)
    return out


def _check_linear(out, x, packed, scale, zp, bias=None):
    group = 2 * packed.size(-1) // scale.size(-1)
    w, x = _dense64(packed, scale, zp, group), x.double()
    y = x @ w.t() + (0 if bias is None else bias.double())
    bound = BF16 * y.abs() * 1.01 + _bf16_off(x) @ w.abs().t() + _gamma(x.size(-1)) * (x.abs() @ w.abs().t() + (0 if bias is None else bias.double().abs()))
    err = (out.double() - y).abs()
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 1, 128), (1, 16, 256), (2, 17, 128), (1, 300, 2048), (3, 33, 384), (8, 64, 1024),
                                   (9, 130, 640), (16, 257, 512), (17, 48, 2048), (31, 100, 896), (33, 65, 256), (70, 40, 384),
                                   (1, 4099, 128), (5, 2048, 4096), (12, 1111, 8192)])
def test_dense_shapes(M, N, K, group):
    g = torch.Generator().manual_seed(M * 1000 + N + K + group)
    zeros = (M + N) % 2 == 1
    w = _weights(N, K, group, zeros, g)
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    bias = torch.randn(N, generator=g).to(torch.bfloat16).cuda() if N % 3 == 0 else None
    _check_linear(_linear(x, *w, bias), x, *w, bias)


@pytest.mark.parametrize("K,group", [(32, 32), (64, 64), (96, 32), (160, 32), (192, 64), (1088, 64), (1184, 32), (4640, 32)])
def test_dense_column_counts_that_fill_no_tile(K, group):
    g = torch.Generator().manual_seed(K)
    for M in (1, 6, 13):
        w = _weights(77, K, group, True, g)
        x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
        _check_linear(_linear(x, *w), x, *w)


def test_every_code_and_zero_point_is_exact():
    """One column at a time: W itself comes back, and (code - zero) * scale fits bf16's roundings exactly for scale 1."""
    codes = torch.arange(16, dtype=torch.uint8).repeat(16, 1)           # row z: codes 0..15
    row = torch.cat([codes, codes.flip(1)], 1)                          # [16, 32]
    packed = (row[:, 0::2] | (row[:, 1::2] << 4)).cuda()
    zero = torch.arange(16, dtype=torch.uint8)[:, None].cuda()
    scale = torch.ones(16, 1, dtype=torch.bfloat16).cuda()
    x = torch.eye(32, dtype=torch.bfloat16).cuda()
    out = _linear(x, packed, scale, zero)
    assert torch.equal(out.t().float().cpu(), row.float() - torch.arange(16.0)[:, None])


def test_leading_dimensions_row_strides_and_empty_batches():
    from layered_prefill_b200 import ops
    g = torch.Generator().manual_seed(3)
    w = _weights(50, 256, 64, False, g)
    x = torch.randn(2, 3, 256, generator=g).to(torch.bfloat16).cuda()
    assert torch.equal(_linear(x, *w).view(6, 50), _linear(x.view(6, 256), *w))
    wide = torch.randn(6, 512, generator=g).to(torch.bfloat16).cuda()
    part = wide[:, 256:]
    assert torch.equal(_linear(part, *w), _linear(part.contiguous(), *w))
    ops.w4_linear(torch.empty(0, 50, dtype=torch.bfloat16, device="cuda"), x.view(6, 256)[:0], *w)


def test_values_of_x_that_are_not_finite_reach_only_their_row():
    g = torch.Generator().manual_seed(4)
    w = _weights(40, 512, 128, True, g)
    x = torch.randn(11, 512, generator=g).to(torch.bfloat16).cuda()
    want = _linear(x, *w)
    bad = x.clone()
    bad[3, 100], bad[9, 0] = float("nan"), float("inf")
    out = _linear(bad, *w)
    rest = [i for i in range(11) if i not in (3, 9)]
    assert torch.equal(out[rest], want[rest])
    assert out[3].isnan().all() and (~out[9].isfinite()).all()


def test_a_row_does_not_depend_on_the_batch_around_it():
    g = torch.Generator().manual_seed(8)
    w = _weights(96, 1024, 64, True, g)
    x = torch.randn(40, 1024, generator=g).to(torch.bfloat16).cuda()
    out = _linear(x, *w)
    for m in (0, 7, 8, 39):
        _check_linear(_linear(x[m:m + 1], *w), x[m:m + 1], *w)
    assert torch.equal(out, _linear(x, *w))  # the same bits twice


# ---------------------------------------------------------------------------------------------------- experts
def _act64(gate, up, activation):
    if activation == "silu":
        return gate * torch.sigmoid(gate) * up
    gate, up = gate.clamp(max=7.0), up.clamp(-7.0, 7.0)
    return gate * torch.sigmoid(1.702 * gate) * (up + 1)


def _experts64(x, w13, w2, b13, b2, tw, ti, group, activation):
    """(out, bound) in 64 bits, slot by slot."""
    T, H = x.shape
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(out)
    E = w13[0].size(0)
    for e in range(E):
        t, j = torch.nonzero(ti == e, as_tuple=True)
        if t.numel() == 0:
            continue
        a = _dense64(w13[0][e], w13[1][e], None if w13[2] is None else w13[2][e], group)
        b = _dense64(w2[0][e], w2[1][e], None if w2[2] is None else w2[2][e], group)
        xe = x[t].double()
        gu = xe @ a.t() + (0 if b13 is None else b13[e].double())
        dgu = _bf16_off(xe) @ a.abs().t() + _gamma(H) * (xe.abs() @ a.abs().t() + (0 if b13 is None else b13[e].double().abs()))
        I = gu.size(1) // 2
        cut = (lambda v: (v[:, :I], v[:, I:])) if activation == "silu" else (lambda v: (v[:, 0::2], v[:, 1::2]))
        (gate, up), (dg, du) = cut(gu), cut(dgu)
        h = _act64(gate, up, activation)
        # slopes: |d act/d gate| <= 1.2 |up + 1|, |d act/d up| <= |gate|
        dh = 1.2 * (up.abs() + 1) * dg + gate.abs() * du + 2.0 ** -20 * gate.abs() * (up.abs() + 1)
        y = h @ b.t() + (0 if b2 is None else b2[e].double())
        dy = (dh + _step(h)) @ b.abs().t() + _gamma(I) * (h.abs() @ b.abs().t() + (0 if b2 is None else b2[e].double().abs()))
        w = tw[t, j].double()[:, None]
        out.index_add_(0, t, w * y)
        bound.index_add_(0, t, w.abs() * dy + 2.0 ** -22 * (w * y).abs())
    return out, bound + 1.01 * BF16 * out.abs()


def _experts(x, w13, w2, tw, ti, group, b13=None, b2=None, activation="silu", inplace=False):
    from layered_prefill_b200 import fused_moe
    return fused_moe.fused_experts(x, w13[0], w2[0], b13, b2, tw, ti, inplace=inplace, activation=activation, w1_scale=w13[1],
                                   w2_scale=w2[1], w1_zp=w13[2], w2_zp=w2[2], block_shape=[0, group])


def _case(T, H, E, k, I, group, zeros, seed, skew=0.0):
    g = torch.Generator().manual_seed(seed)
    w13 = _weights(2 * I, H, group, zeros, g, (E,))
    w2 = _weights(H, I, group, zeros, g, (E,))
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).cuda()
    tw, ti = torch.topk(torch.softmax(torch.randn(T, E, generator=g) + skew * torch.randn(E, generator=g), -1), k, -1)
    return x, w13, w2, tw.cuda(), ti.to(torch.int32).cuda()


def _check_experts(out, *args):
    want, bound = _experts64(*args)
    err = (out.double() - want).abs()
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("T,H,E,k,I,group", [
    (1, 128, 8, 1, 64, 32), (1, 2048, 128, 8, 768, 128), (2, 256, 8, 2, 128, 128), (3, 512, 4, 4, 96, 32),
    (7, 640, 16, 6, 192, 64), (17, 256, 60, 4, 160, 32), (64, 256, 16, 8, 128, 64), (64, 1024, 128, 8, 256, 128),
    (100, 384, 8, 8, 256, 128), (200, 128, 8, 2, 64, 64), (33, 4096, 8, 2, 1536, 128), (9, 192, 3, 3, 64, 64), (5, 96, 8, 2, 32, 32)])
@pytest.mark.parametrize("zeros", [False, True])
def test_expert_shapes(T, H, E, k, I, group, zeros):
    x, w13, w2, tw, ti = _case(T, H, E, k, I, group, zeros, T + H + I)
    _check_experts(_experts(x, w13, w2, tw, ti, group), x, w13, w2, None, None, tw, ti, group, "silu")


@pytest.mark.parametrize("T", [1, 20, 150])
def test_interleaved_activation_and_biases(T):
    x, w13, w2, tw, ti = _case(T, 256, 8, 2, 128, 64, True, 5 + T)
    g = torch.Generator().manual_seed(1)
    b13 = torch.randn(8, 256, generator=g).to(torch.bfloat16).cuda()
    b2 = torch.randn(8, 256, generator=g).to(torch.bfloat16).cuda()
    for act in ("swigluoai", "silu"):
        _check_experts(_experts(x, w13, w2, tw, ti, 64, b13, b2, act), x, w13, w2, b13, b2, tw, ti, 64, act)


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("act", ["silu", "swigluoai"])
def test_values_that_are_not_finite_reach_their_token_through_the_experts(T, act):
    x, w13, w2, tw, ti = _case(T, 256, 8, 2, 128, 64, True, 12)
    want = _experts(x, w13, w2, tw, ti, 64, None, None, act)
    for value in (float("nan"), float("inf"), float("-inf")):
        bad = x.clone()
        bad[1, 77] = value
        out = _experts(bad, w13, w2, tw, ti, 64, None, None, act)
        assert out[1].isnan().all()
        rest = [t for t in range(T) if t != 1]
        assert torch.equal(out[rest], want[rest])


def test_one_expert_takes_every_token():
    x, w13, w2, tw, ti = _case(90, 256, 8, 1, 128, 32, False, 2)
    ti[:] = 5
    _check_experts(_experts(x, w13, w2, tw, ti, 32), x, w13, w2, None, None, tw, ti, 32, "silu")


def test_the_same_expert_twice_and_slots_without_one():
    x, w13, w2, tw, ti = _case(12, 256, 8, 4, 128, 64, True, 3)
    ti[:, 1] = ti[:, 0]          # the same expert twice for every token
    ti[2, :] = -1                # a token without an expert
    ti[4, 3] = 8                 # outside
    ti[5, 0] = -7
    out = _experts(x, w13, w2, tw, ti, 64)
    _check_experts(out, x, w13, w2, None, None, tw, ti, 64, "silu")
    assert (out[2] == 0).all()
    ti[:] = -1
    assert (_experts(x, w13, w2, tw, ti, 64) == 0).all()


def test_in_place_empty_batch_and_other_index_types():
    x, w13, w2, tw, ti = _case(10, 256, 8, 2, 128, 128, False, 4)
    want = _experts(x, w13, w2, tw, ti, 128)
    assert torch.equal(_experts(x, w13, w2, tw, ti.long(), 128), want)
    y = x.clone()
    assert _experts(y, w13, w2, tw, ti, 128, inplace=True).data_ptr() == y.data_ptr()
    assert torch.equal(y, want)
    assert _experts(x[:0], w13, w2, tw[:0], ti[:0], 128).shape == (0, 256)


def test_experts_on_two_streams_at_once_and_in_two_graphs():
    a, b = (_case(24, 512, 16, 4, 256, 64, True, s) for s in (21, 22))
    want = [_experts(*c[:3], c[3], c[4], 64) for c in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(20):
        for i, c in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i] = _experts(*c[:3], c[3], c[4], 64)
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(want, got))
    graphs, outs = [], []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_experts(*c[:3], c[3], c[4], 64))
        graphs.append(g)
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(want, outs))


def test_quantised_weights_come_near_the_bf16_block():
    """A run of the operators as they are used: quant_w4 once, then norm -> router -> 4-bit experts -> 4-bit projection."""
    from layered_prefill_b200 import fused_moe, linear, ops
    T, H, E, k, I, g = 24, 512, 16, 4, 256, 64
    gen = torch.Generator().manual_seed(2)
    w13 = (torch.randn(E, 2 * I, H, generator=gen) * 0.05).cuda()
    w2 = (torch.randn(E, H, I, generator=gen) * 0.05).cuda()
    wg = (torch.randn(E, H, generator=gen) * 0.05).to(torch.bfloat16).cuda()
    wo = torch.randn(H, 2 * H, generator=gen) * 0.05
    q13, q2 = fused_moe.quant_w4(w13, g, True), fused_moe.quant_w4(w2, g, True)
    attn = torch.randn(T, 2 * H, generator=gen).to(torch.bfloat16).cuda()
    residual = torch.randn(T, H, generator=gen).to(torch.bfloat16).cuda()
    o_proj = linear.W4RowParallelLinear(2 * H, H, group_size=g, zero_points=True)
    for name, value in zip(("qweight", "scales", "zeros"), fused_moe.quant_w4(wo, g, True)):
        p = getattr(o_proj, name)
        p.weight_loader(p, value)
    o_proj = o_proj.cuda()
    y = o_proj(attn)
    _check_linear(y, attn, o_proj.qweight, o_proj.scales, o_proj.zeros)
    norm_w = torch.ones(H, dtype=torch.bfloat16, device="cuda")
    normed, new_res = o_proj.forward_reduce_norm(attn, residual.clone(), norm_w, 1e-6)
    q = torch.empty(T, H, dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty(T, H // 128, device="cuda")
    hidden = torch.empty_like(residual)
    ops.add_rms_norm_quant_fp8(q, s, residual, y, norm_w, 1e-6, normed_out=hidden)
    assert torch.equal(residual, new_res)
    logits = hidden @ wg.t()
    tw, ti, balance, z, counts = fused_moe.fused_topk_with_loss(logits, k, True)
    assert int(counts.sum()) == T * k and float(balance) >= 0.99 * k
    got = fused_moe.fused_moe_forward_w4(hidden, logits, q13, q2, k, g)
    _check_experts(got, hidden, q13, q2, None, None, tw, ti, g, "silu")
    ref = fused_moe.fused_experts(hidden, w13.to(torch.bfloat16), w2.to(torch.bfloat16), None, None, tw, ti)
    # each code is off by at most half a step of a range of 15 steps: with random errors 2 * sqrt(1/12) / (15 / 5.6) ~ 0.11 a matrix
    assert (got.float() - ref.float()).norm() / ref.float().norm() < 0.3


@pytest.mark.parametrize("M,N,K,group", [(3, 40, 16384, 128), (16, 100, 16384, 64), (24, 70, 8192, 32), (40, 300, 4096, 128)])
def test_dense_columns_that_do_not_fit_at_once(M, N, K, group):
    g = torch.Generator().manual_seed(M + K)
    w = _weights(N, K, group, True, g)
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    _check_linear(_linear(x, *w), x, *w)


@pytest.mark.parametrize("M", [2, 20])
def test_outliers_next_to_small_values(M):
    """A few columns thousands of times larger than the rest, rows of zeros, and the ends of the range of bf16."""
    g = torch.Generator().manual_seed(12)
    w = _weights(64, 2048, 64, True, g)
    x = torch.randn(M, 2048, generator=g)
    x[:, ::257] *= 3000
    x[0, 128:256] = 0
    x[1, 256:384] *= 2.0 ** -100
    x[1, 384:512] *= 2.0 ** 60
    x = x.to(torch.bfloat16).cuda()
    _check_linear(_linear(x, *w), x, *w)
    assert (_linear(torch.zeros_like(x), *w) == 0).all()
    tiny = torch.full_like(x, 2.0 ** -130)
    assert (_linear(tiny, *w).abs() <= 2.0 ** -100).all()
    huge = torch.zeros_like(x)
    huge[:, 5] = 2.0 ** 126
    _check_linear(_linear(huge, *w), huge, *w)


@pytest.mark.parametrize("T,H,E,k,I,group", [(300, 256, 16, 8, 64, 32), (1030, 128, 8, 1, 64, 64), (9, 8192, 4, 2, 128, 128),
                                             (12, 128, 4, 2, 6400, 128), (5, 10240, 3, 2, 96, 32), (64, 256, 200, 6, 64, 32)])
def test_experts_in_pieces_and_with_long_columns(T, H, E, k, I, group):
    """More slots than are listed at once, activations that do not fit at once, more experts than slots of a token."""
    x, w13, w2, tw, ti = _case(T, H, E, k, I, group, True, T + H)
    _check_experts(_experts(x, w13, w2, tw, ti, group), x, w13, w2, None, None, tw, ti, group, "silu")
    if T == 300:
        want = _experts(x, w13, w2, tw, ti, group)
        y = x.clone()
        _experts(y, w13, w2, tw, ti, group, inplace=True)
        assert torch.equal(y, want)


def test_on_scales_and_codes_between_the_usual_boundaries():
    """Scales and zero points two bytes and one byte off: read one at a time. Codes off sixteen bytes are refused."""
    from layered_prefill_b200._lib import MoeB200Error
    g = torch.Generator().manual_seed(6)
    q, s, z = _weights(48, 1024, 32, True, g)
    x = torch.randn(10, 1024, generator=g).to(torch.bfloat16).cuda()
    want = _linear(x, q, s, z)
    s2 = torch.empty(s.numel() + 1, dtype=s.dtype, device="cuda")[1:].view_as(s).copy_(s)
    z2 = torch.empty(z.numel() + 1, dtype=z.dtype, device="cuda")[1:].view_as(z).copy_(z)
    assert torch.equal(_linear(x, q, s2, z2), want)
    q2 = torch.empty(q.numel() + 8, dtype=q.dtype, device="cuda")[8:].view_as(q).copy_(q)
    with pytest.raises(MoeB200Error):
        _linear(x, q2, s, z)


def _big(shape_n, k, group, lead, g):
    packed = torch.randint(0, 256, (*lead, shape_n, k // 2), generator=g, dtype=torch.uint8, device="cuda")
    scale = (0.01 + 0.02 * torch.rand(*lead, shape_n, k // group, generator=g, device="cuda")).to(torch.bfloat16)
    return packed, scale, None


def test_dense_codes_past_32_bits():
    g = torch.Generator(device="cuda").manual_seed(3)
    N, K = 2**20 + 1003, 8192  # 4096 bytes a row: the last 1003 rows lie past 2^32 bytes
    packed, scale, _ = _big(N, K, 128, (), g)
    x = torch.randn(2, K, generator=g, device="cuda").to(torch.bfloat16)
    out = _linear(x, packed, scale, None)
    for lo, hi in ((0, 40), (2**19 - 20, 2**19 + 20), (2**20 - 20, 2**20 + 20), (N - 40, N)):
        _check_linear(out[:, lo:hi], x, packed[lo:hi], scale[lo:hi], None)


def test_as_many_experts_as_may_be_with_codes_past_32_bits():
    g = torch.Generator(device="cuda").manual_seed(6)
    E, H, I = 1024, 8192, 1024
    w13, w2 = _big(2 * I, H, 128, (E,), g), _big(H, I, 128, (E,), g)
    x = torch.randn(3, H, generator=g, device="cuda").to(torch.bfloat16)
    ti = torch.tensor([[0, 1023, 511, 900], [1023, 512, 1, 700], [1022, 1023, 600, 513]], dtype=torch.int32, device="cuda")
    tw = torch.rand(3, 4, generator=g, device="cuda")
    _check_experts(_experts(x, w13, w2, tw, ti, 128), x, w13, w2, None, None, tw, ti, 128, "silu")


def test_as_many_slots_a_token_as_may_be():
    x, w13, w2, _, _ = _case(2, 128, 1024, 1, 32, 32, False, 15)
    g = torch.Generator().manual_seed(15)
    ti = torch.stack([torch.randperm(1024, generator=g) for _ in range(2)]).to(torch.int32).cuda()
    tw = torch.rand(2, 1024, generator=g).cuda()
    out = _experts(x, w13, w2, tw, ti, 32)
    want, bound = _experts64(x, w13, w2, None, None, tw, ti, 32, "silu")
    # 1024 slots in a row of fp32 additions: a rounding each of at most the sum of the magnitudes
    w13d, w2d = _dense64(*w13, 32), _dense64(*w2, 32)
    gate, up = torch.einsum("th,enh->ten", x.double(), w13d).chunk(2, -1)
    y = torch.einsum("ten,ehn->teh", _act64(gate, up, "silu"), w2d)
    sizes = (y.abs() * tw.double().gather(1, ti.long().argsort(1))[..., None]).sum(1)
    err = (out.double() - want).abs()
    assert (err <= bound + 1024 * 2.0 ** -24 * sizes).all()


def test_dense_on_two_streams_at_once_and_in_a_graph():
    g = torch.Generator().manual_seed(14)
    w = _weights(2048, 4096, 128, False, g)
    xs = [torch.randn(m, 4096, generator=g).to(torch.bfloat16).cuda() for m in (1, 16)]
    want = [_linear(x, *w) for x in xs]
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = _linear(xs[i], *w)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _linear(xs[1], *w)
    keep = xs[1].clone()
    xs[1].zero_()
    graph.replay()
    assert (out == 0).all()
    xs[1].copy_(keep)
    graph.replay()
    assert torch.equal(out, want[1])


def test_refusals():
    from layered_prefill_b200 import fused_moe, ops
    from layered_prefill_b200._lib import MoeB200Error
    g = torch.Generator().manual_seed(1)
    q, s, z = _weights(32, 256, 64, True, g)
    x = torch.randn(4, 256, generator=g).to(torch.bfloat16).cuda()
    out = torch.empty(4, 32, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(input=x[:, :128]), dict(input=x.float()), dict(out=out[:3]), dict(qweight=q.t().contiguous().t()),
                dict(scales=s.float()), dict(zeros=z[:, :1]), dict(zeros=z.cpu()), dict(bias=s[0]), dict(input=x.t())):
        kw = {**dict(out=out, input=x, qweight=q, scales=s, zeros=z), **bad}
        with pytest.raises(RuntimeError):
            ops.w4_linear(**kw)
    with pytest.raises(MoeB200Error):  # groups of 256
        ops.w4_linear(out, x, q, s[:, :1].contiguous())
    with pytest.raises(MoeB200Error):  # a row stride that breaks 16-byte rows
        ops.w4_linear(out, torch.empty(4, 260, dtype=torch.bfloat16, device="cuda")[:, :256], q, s)
    with pytest.raises(MoeB200Error):  # rows on top of each other
        ops.w4_linear(out, x[:1].expand(4, 256), q, s)
    with pytest.raises(MoeB200Error):  # a start between 16-byte boundaries
        ops.w4_linear(out[:1], torch.empty(264, dtype=torch.bfloat16, device="cuda")[1:257].view(1, 256), q, s)
    x, w13, w2, tw, ti = _case(4, 256, 8, 2, 128, 64, True, 1)
    good = dict(w1_scale=w13[1], w2_scale=w2[1], w1_zp=w13[2], w2_zp=w2[2], block_shape=[0, 64])
    for bad in (dict(w1_scale=None), dict(w1_zp=None), dict(block_shape=[0, 48]), dict(block_shape=[0, 128]),
                dict(w1_scale=w13[1].float()), dict(a1_scale=tw), dict(expert_map=ti), dict(activation="gelu"),
                dict(apply_router_weight_on_input=True), dict(w2_scale=w2[1][:, :, :1])):
        with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
            fused_moe.fused_experts(x, w13[0], w2[0], None, None, tw, ti, **{**good, **bad})
    with pytest.raises(RuntimeError):
        fused_moe.fused_experts(x.float(), w13[0], w2[0], None, None, tw, ti, **good)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_weights_of_zero_give_zero(group, zeros):
    """Codes equal to their zero points, scales that are not zero, activations of one sign and of many magnitudes."""
    g = torch.Generator().manual_seed(group)
    N, K = 48, 640
    zp = torch.randint(9, 16, (N, K // group), generator=g, dtype=torch.uint8) if zeros else torch.full((N, K // group), 8, dtype=torch.uint8)
    code = zp.repeat_interleave(group, 1)
    packed = (code[:, 0::2] | (code[:, 1::2] << 4)).cuda()
    scale = torch.rand(N, K // group, generator=g).add(0.5).to(torch.bfloat16).cuda()
    for M in (1, 7, 16, 40):
        x = (torch.rand(M, K, generator=g) * 2.0 ** torch.randint(-6, 1, (M, K), generator=g)).to(torch.bfloat16).cuda()
        assert (_linear(x, packed, scale, zp.cuda() if zeros else None) == 0).all()
    I = 128
    x, w13, _, tw, ti = _case(9, 128, 4, 2, I, group, zeros, 3)
    zp = zp[:, :1].repeat(3, I // group)[:128]
    code = zp.repeat_interleave(group, 1)
    w2 = (code[:, 0::2] | (code[:, 1::2] << 4)).expand(4, 128, I // 2).contiguous().cuda()
    s2 = torch.ones(4, 128, I // group, dtype=torch.bfloat16, device="cuda")
    z2 = zp.expand(4, 128, I // group).contiguous().cuda() if zeros else None
    assert (_experts(x, w13, (w2, s2, z2), tw, ti, group) == 0).all()


@pytest.mark.parametrize("M", [1, 19])
def test_row_parallel_linear_with_a_bias_under_the_default_type(M):
    from layered_prefill_b200 import fused_moe, linear, ops
    assert torch.get_default_dtype() == torch.float32
    g = torch.Generator().manual_seed(M)
    N, K = 256, 512
    layer = linear.W4RowParallelLinear(K, N, bias=True, group_size=64)
    for name, value in zip(("qweight", "scales"), fused_moe.quant_w4(torch.randn(N, K, generator=g) * 0.05, 64)):
        p = getattr(layer, name)
        p.weight_loader(p, value)
    layer.bias.weight_loader(layer.bias, torch.randn(N, generator=g))
    layer = layer.cuda()
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).cuda()
    y = layer(x)
    _check_linear(y, x, layer.qweight, layer.scales, None, layer.bias)
    residual = torch.randn(M, N, generator=g).to(torch.bfloat16).cuda()
    norm_w = torch.rand(N, generator=g).to(torch.bfloat16).cuda()
    normed, res = layer.forward_reduce_norm(x, residual.clone(), norm_w, 1e-6)
    want = torch.empty_like(y)
    ops.add_rms_norm(want, residual, y, norm_w, 1e-6)
    assert torch.equal(normed, want) and torch.equal(res, residual)


# ------------------------------------------------------------------------- small values next to large ones
# Where the integers would cut off too much of 128 columns (the sum of min(|x| / f, 1024)^2 is below 2^24, f being the step, 2^-14 of the power
# of two at or below the largest) what they cut off is added as further integers in steps of 2^-15 f: off by half of one, or by a whole one where the
# largest rounds up, so by at most 2^-15 f <= 2^-29 of the largest. The step of such columns carries a mark in its last bit, which moves
# their products by 2^-23, as one more of the 64 further additions does.
def _cut(x, unmarked):
    """What x [.., K] may be off by: 2^-29 of the largest in marked columns, unmarked(x) in the others."""
    K = x.size(-1)
    v = torch.nn.functional.pad(x.double(), (0, -K % 128)).unflatten(-1, (-1, 128))
    big = v.abs().amax(-1, keepdim=True)
    f = torch.where(big > 0, torch.exp2(torch.floor(torch.log2(big.clamp(min=2.0 ** -120))) - 14), torch.ones_like(big))
    few = ((v / f).abs().clamp(max=1024).square().sum(-1, keepdim=True) < 2.0 ** 24).expand_as(v).flatten(-2)[..., :K]
    return torch.where(few, 2.0 ** -29 * big.expand_as(v).flatten(-2)[..., :K], unmarked(x.double()))


def _ignoring(packed, zp, group, columns):
    """The codes with those of some columns equal to their zero points."""
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    z = torch.full_like(code, 8) if zp is None else zp.repeat_interleave(group, -1)
    code[..., columns] = z[..., columns]
    return code[..., 0::2] | (code[..., 1::2] << 4)


@pytest.mark.parametrize("factor", [100.0, 3000.0, 1e6])
@pytest.mark.parametrize("M,N,K,group,zeros", [(1, 64, 2048, 128, False), (3, 70, 640, 32, True), (8, 33, 1024, 64, True), (16, 128, 2048, 128, True),
                                               (20, 64, 8192, 64, False), (7, 2400, 2048, 32, False), (16, 100, 16384, 64, True),
                                               (5, 17, 96, 32, True), (40, 4096, 512, 128, False)])
def test_small_values_next_to_large_ones_that_a_row_ignores(M, N, K, group, zeros, factor):
    """A few columns far larger than the rest; half of the rows have no weight for them."""
    g = torch.Generator().manual_seed(M + N + K)
    packed, scale, zp = _weights(N, K, group, zeros, g)
    large = torch.arange(5, K, 64)
    packed[: N // 2] = _ignoring(packed[: N // 2].clone(), None if zp is None else zp[: N // 2], group, large.cuda())
    x = torch.randn(M, K, generator=g)
    x[:, large] = factor * (1 + torch.rand(M, large.numel(), generator=g))
    x = x.to(torch.bfloat16).cuda()
    out = _linear(x, packed, scale, zp)
    w, xd = _dense64(packed, scale, zp, group), x.double()
    y = xd @ w.t()
    bound = 1.01 * BF16 * y.abs() + _cut(x, _bf16_off) @ w.abs().t() + _gamma(K) * (xd.abs() @ w.abs().t())
    err = (out.double() - y).abs()
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("T,act,zeros", [(1, "silu", True), (6, "silu", False), (21, "swigluoai", True), (1030, "silu", True)])
def test_small_intermediates_next_to_large_ones_that_a_row_ignores(T, act, zeros):
    """The same in both products of the experts: hidden states and the activations between, which are fp32."""
    g = torch.Generator().manual_seed(T)
    H, I, group = 512, 256, 64
    w13, w2 = _weights(2 * I, H, group, zeros, g, (1,)), _weights(H, I, group, zeros, g, (1,))
    large_x, large_h = torch.arange(7, H, 128).cuda(), torch.arange(3, I, 128).cuda()
    keep = w13[0].clone()
    w13 = (_ignoring(w13[0].clone(), w13[2], group, large_x), w13[1], w13[2])
    for i in large_h.tolist():  # these columns between the products do see the large hidden states: they come out large
        rows = [i, I + i] if act == "silu" else [2 * i + 1]
        w13[0][:, rows] = keep[:, rows]
    w2 = (_ignoring(w2[0].clone(), w2[2], group, large_h), w2[1], w2[2])
    x = torch.randn(T, H, generator=g)
    x[:, large_x.cpu()] = 2000.0
    x = x.to(torch.bfloat16).cuda()
    tw, ti = torch.ones(T, 1, device="cuda"), torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    out = _experts(x, w13, w2, tw, ti, group, activation=act)
    a, b, xd = _dense64(*(t if t is None else t[0] for t in w13), group), _dense64(*(t if t is None else t[0] for t in w2), group), x.double()
    gu, dgu = xd @ a.t(), _cut(x, _bf16_off) @ a.abs().t() + _gamma(H) * (xd.abs() @ a.abs().t())
    cut = (lambda v: (v[:, :I], v[:, I:])) if act == "silu" else (lambda v: (v[:, 0::2], v[:, 1::2]))
    (gate, up), (dg, du) = cut(gu), cut(dgu)
    h = _act64(gate, up, act)
    dh = 1.2 * (up.abs() + 1) * dg + gate.abs() * du + 2.0 ** -20 * gate.abs() * (up.abs() + 1)
    y = h @ b.t()
    bound = 1.01 * BF16 * y.abs() + (dh + _cut(h, _step)) @ b.abs().t() + _gamma(I) * (h.abs() @ b.abs().t())
    err = (out.double() - y).abs()
    assert (err <= bound).all(), (err / bound).max()


def test_marked_activations_prepared_in_front_or_by_each_block_give_the_same_bits():
    from layered_prefill_b200 import ops
    from layered_prefill_b200._lib import lib
    g = torch.Generator().manual_seed(5)
    M, N, K, group = 13, 200, 2048, 64
    packed, scale, zp = _weights(N, K, group, True, g)
    x = torch.randn(M, K, generator=g)
    x[:, 9::200] = 900.0
    x[4] = torch.randn(K, generator=g)  # a token without large columns between those with
    x = x.to(torch.bfloat16).cuda()
    with_room = _linear(x, packed, scale, zp)
    assert lib.moe_b200_w4_linear_workspace_bytes(M, K, group) > 0
    out = torch.empty_like(with_room)
    ops._launch(lib.moe_b200_w4_linear, out.device, out.data_ptr(), x.data_ptr(), K, packed.data_ptr(), scale.data_ptr(), zp.data_ptr(), 0, M, N,
                K, group, 0, 0)
    assert torch.equal(out, with_room)
    bad = x.clone()
    bad[2, 9], bad[5, 0], bad[7, 700] = float("inf"), float("nan"), float("-inf")
    out = _linear(bad, packed, scale, zp)
    rest = [i for i in range(M) if i not in (2, 5, 7)]
    assert out[[2, 5, 7]].isnan().all() and torch.equal(out[rest], with_room[rest])


def test_marked_activations_of_strided_rows_and_in_a_graph():
    g = torch.Generator().manual_seed(9)
    N, K, group = 96, 1024, 32
    packed, scale, zp = _weights(N, K, group, True, g)
    wide = torch.randn(9, 2 * K, generator=g)
    wide[:, K + 3::170] = 4000.0
    wide = wide.to(torch.bfloat16).cuda()
    part = wide[:, K:]
    want = _linear(part.contiguous(), packed, scale, zp)
    assert torch.equal(_linear(part, packed, scale, zp), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _linear(part, packed, scale, zp)
    keep = wide.clone()
    wide.copy_(torch.randn(9, 2 * K, generator=g))  # nothing stands out: no marks
    graph.replay()
    assert torch.equal(out, _linear(part.contiguous(), packed, scale, zp)) and not torch.equal(out, want)
    wide.copy_(keep)
    graph.replay()
    assert torch.equal(out, want)
