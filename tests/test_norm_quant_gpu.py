"""(add +) RMS norm with an e4m3 output, against the same operator in 64 bits.

Tolerances. y is computed in fp32: the mean of H squares is a chain of at most 32 fused multiply-adds and ten shuffled adds,
rsqrt and two products, together under 64 roundings of 2^-24, so |dy| <= 2^-18 |y|. An e4m3 code is off by half a step: 2^-4 of the
value, or half of the smallest step (2^-10 scales) below the normal range; bf16 outputs by 2^-8 of the value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FP32 = 2.0 ** -18
BF16 = 2.0 ** -8
E4M3 = 2.0 ** -4


def _inputs(T, H, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, H, generator=g) * scale).to(torch.bfloat16).cuda()
    res = (3 * torch.randn(T, H, generator=g)).to(torch.bfloat16).cuda()
    w = (1 + 0.2 * torch.randn(H, generator=g)).to(torch.bfloat16).cuda()
    return x, res, w


def _oracle(r, w, eps, group):
    r = r.double()
    y = r / torch.sqrt(r.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    width = r.size(-1) if group == -1 else group
    s = y.unflatten(-1, (-1, width)).abs().amax(-1).clamp(min=1e-10) / 448
    return y, s, s.repeat_interleave(width, -1)


def _run(x, res, w, group, normed, in_place=False, eps=1e-6):
    from layered_prefill_b200 import ops
    T, H = x.shape
    q = torch.empty(T, H, dtype=torch.float8_e4m3fn, device=x.device)
    s = torch.empty(T, 1 if group == -1 else H // 128, dtype=torch.float32, device=x.device)
    n = torch.empty_like(x) if normed else None
    if res is None:
        ops.rms_norm_quant_fp8(q, s, x, w, eps, group_size=group, normed_out=n)
        return q, s, n, x
    out = res.clone() if in_place else torch.empty_like(res)
    if in_place:
        ops.add_rms_norm_quant_fp8(q, s, out, x, w, eps, group_size=group, normed_out=n)
    else:
        kept = res.clone()
        ops.add_rms_norm_quant_fp8(q, s, res, x, w, eps, group_size=group, normed_out=n, residual_out=out)
        assert torch.equal(res, kept)
    return q, s, n, out


def _check(q, s, n, r, w, group, eps=1e-6):
    y, s64, wide = _oracle(r, w, eps, group)
    assert ((s.double() - s64).abs() <= FP32 * s64).all()
    back = q.double() * s.double().repeat_interleave(q.size(-1) // s.size(-1), -1)
    assert ((back - y).abs() <= (E4M3 + 2 * FP32) * y.abs() + wide * 2.0 ** -10 * (1 + FP32)).all()
    if n is not None:
        assert ((n.double() - y).abs() <= (BF16 + FP32) * y.abs()).all()


@pytest.mark.parametrize("T,H", [(1, 128), (1, 2048), (3, 384), (64, 2048), (130, 4096), (5, 1152), (2, 16384), (2, 32768)])
@pytest.mark.parametrize("residual", [False, True])
def test_groups_of_128(T, H, residual):
    x, res, w = _inputs(T, H, T + H)
    q, s, n, r = _run(x, res if residual else None, w, 128, True)
    if residual:
        assert torch.equal(r, (x.float() + res.float()).to(torch.bfloat16))
    _check(q, s, n, r, w, 128)


@pytest.mark.parametrize("T,H", [(1, 8), (7, 24), (2, 128), (65, 1000), (3, 5000), (33, 2056), (2, 24008), (1, 32760)])
@pytest.mark.parametrize("residual", [False, True])
def test_one_scale_a_token(T, H, residual):
    x, res, w = _inputs(T, H, 7 * T + H)
    q, s, n, r = _run(x, res if residual else None, w, -1, False)
    if residual:
        assert torch.equal(r, (x.float() + res.float()).to(torch.bfloat16))
    _check(q, s, n, r, w, -1)


@pytest.mark.parametrize("H", [12288, 12296, 32768])
def test_where_a_thread_takes_more_vectors(H):
    x, res, w = _inputs(3, H, H)
    for group in (128, -1) if H % 128 == 0 else (-1,):
        q, s, n, r = _run(x, res, w, group, True)
        _check(q, s, n, r, w, group)


def test_residual_in_place_and_the_same_bits_twice():
    x, res, w = _inputs(40, 2048, 5)
    a, b = _run(x, res, w, 128, True), _run(x, res, w, 128, True, in_place=True)
    for u, v in zip(a, b):
        assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))


def test_agrees_with_the_norm_and_the_quantisation_it_joins():
    """add_rms_norm rounds twice to bf16 before the quantisation: three half steps of bf16 and two of e4m3 apart at most."""
    from layered_prefill_b200 import fused_moe, ops
    x, res, w = _inputs(64, 2048, 6)
    q, s, n, r = _run(x, res, w, 128, True)
    normed, res2 = torch.empty_like(x), res.clone()
    ops.add_rms_norm(normed, res2, x, w, 1e-6)
    assert torch.equal(r, res2)
    assert ((normed.double() - n.double()).abs() <= 3.1 * BF16 * n.double().abs()).all()
    q2, s2 = fused_moe.per_token_group_quant_fp8(normed)
    assert ((s - s2).abs() <= 2.1 * BF16 * s).all()
    a, b = (u.double() * v.double().repeat_interleave(128, -1) for u, v in ((q, s), (q2, s2)))
    assert ((a - b).abs() <= (2 * E4M3 + 5 * BF16) * a.abs().maximum(b.abs()) + s.double().repeat_interleave(128, -1) * 2.0 ** -9 * 1.1).all()


def test_zero_rows_outliers_and_nan():
    x, _, w = _inputs(6, 256, 9)
    x[1] = 0                      # the scale stays at its floor, the codes are zero
    x[2, 7] = 30000.0             # one outlier sets its group's scale
    x[3] = torch.finfo(torch.bfloat16).tiny
    x[4, 130] = float("nan")      # the mean is NaN: the whole token is
    q, s, n, r = _run(x, None, w, 128, True)
    ok = [0, 1, 2, 3, 5]
    _check(q[ok], s[ok], n[ok], r[ok], w, 128)
    assert (q[1].float() == 0).all() and torch.allclose(s[1], torch.full_like(s[1], 1e-10 / 448), rtol=1e-6)
    assert s[4].isnan().all() and q[4].float().isnan().all() and n[4].isnan().all()
    x[4, 130] = float("inf")      # inf * rsqrt(inf) is NaN there, the others become zero
    q, s, n, _ = _run(x, None, w, 128, True)
    assert s[4, 1].isnan() and n[4, 130].isnan() and (n[4, :128] == 0).all()


def test_rows_past_the_batch_stay_and_leading_dimensions():
    from layered_prefill_b200 import ops
    x, res, w = _inputs(12, 512, 4)
    q = torch.full((14, 512), 3.0, device="cuda").to(torch.float8_e4m3fn)
    s = torch.full((14, 4), -1.0, device="cuda")
    ops.rms_norm_quant_fp8(q[:12].view(3, 4, 512), s[:12].view(3, 4, 4), x.view(3, 4, 512), w, 1e-6)
    assert (q[12:].float() == 3).all() and (s[12:] == -1).all()
    _check(q[:12], s[:12], None, x, w, 128)
    ops.rms_norm_quant_fp8(q[:0], s[:0], x[:0], w, 1e-6)  # no token


def test_offsets_past_32_bits():
    g = torch.Generator(device="cuda").manual_seed(2)
    T, H = 2**18 + 70, 16384
    x = torch.randn(T, H, generator=g, device="cuda", dtype=torch.bfloat16)
    w = (1 + 0.2 * torch.randn(H, generator=g, device="cuda")).to(torch.bfloat16)
    q, s, n, _ = _run(x, None, w, 128, True)
    for lo, hi in ((0, 9), (2**17 - 4, 2**17 + 4), (2**18 - 4, 2**18 + 4), (T - 9, T)):
        _check(q[lo:hi], s[lo:hi], n[lo:hi], x[lo:hi], w, 128)


def test_on_another_stream_and_in_a_graph():
    from layered_prefill_b200 import ops
    x, res, w = _inputs(33, 1024, 3)
    want = _run(x, res, w, 128, True)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = _run(x, res, w, 128, True)
    torch.cuda.current_stream().wait_stream(st)
    for u, v in zip(want, got):
        assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))
    q, s, n, r = (torch.empty_like(t) for t in want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.add_rms_norm_quant_fp8(q, s, res, x, w, 1e-6, normed_out=n, residual_out=r)
    x.neg_()
    g.replay()
    torch.cuda.synchronize()
    _check(q, s, n, (x.float() + res.float()).to(torch.bfloat16), w, 128)


def test_feeds_the_e4m3_experts():
    """The experts on (codes, scales) equal the experts that quantise the same values themselves, where the values are exact."""
    from layered_prefill_b200 import fused_moe, ops
    from oracle import moe_oracle as O
    T, H, E, k, I = 20, 256, 8, 2, 128
    g = torch.Generator().manual_seed(1)
    x, res, w = _inputs(T, H, 2)
    w13 = (torch.randn(E, 2 * I, H, generator=g) * 0.05).to(torch.bfloat16)
    w2 = (torch.randn(E, H, I, generator=g) * 0.05).to(torch.bfloat16)
    (q13, s13), (q2, s2) = O.quant_weight_block_fp8(w13), O.quant_weight_block_fp8(w2)
    q13, s13, q2, s2 = (t.cuda() for t in (q13, s13, q2, s2))
    tw, ti, _ = fused_moe.fused_topk(x, torch.randn(T, E, generator=g).cuda(), k, True)
    q, s, n, _ = _run(x, res, w, 128, True)
    kw = dict(w1_scale=s13, w2_scale=s2, block_shape=[128, 128])
    got = fused_moe.fused_experts(q, q13, q2, None, None, tw, ti, a1_scale=s, **kw)
    assert got.dtype == torch.bfloat16
    # the same codes through the quantising entry: bf16 activations whose quantisation gives those codes back exactly
    qb, sb = fused_moe.per_token_group_quant_fp8(n)
    want = fused_moe.fused_experts(n, q13, q2, None, None, tw, ti, **kw)
    again = fused_moe.fused_experts(qb, q13, q2, None, None, tw, ti, a1_scale=sb, **kw)
    assert torch.equal(want, again)
    # from the unrounded norm: other roundings of the same activations (e4m3 half steps, random)
    rel = (got.float() - want.float()).norm() / want.float().norm()
    assert rel < 2 * E4M3
    with pytest.raises(ValueError):
        fused_moe.fused_experts(q, q13, q2, None, None, tw, ti, **kw)
    with pytest.raises(NotImplementedError):
        fused_moe.fused_experts(q, q13, q2, None, None, tw, ti, a1_scale=s, inplace=True, **kw)
    assert ops.read_status(torch.device("cuda", 0)) == 0


def test_refusals():
    from layered_prefill_b200 import ops
    from layered_prefill_b200._lib import MoeB200Error
    x, res, w = _inputs(4, 256, 1)
    q = torch.empty(4, 256, dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty(4, 2, device="cuda")
    for bad in (dict(out=q[:3]), dict(out=q.view(torch.uint8)), dict(scales=s[:, :1]), dict(scales=s.double()),
                dict(input=x.t().contiguous().t()), dict(input=x.float()), dict(weight=w[:-8]), dict(input=x.cpu())):
        kw = {**dict(out=q, scales=s, input=x, weight=w, epsilon=1e-6), **bad}
        with pytest.raises(RuntimeError):
            ops.rms_norm_quant_fp8(**kw)
    with pytest.raises(MoeB200Error):
        ops.rms_norm_quant_fp8(q, s, x, w, 1e-6, group_size=64)
    off = torch.empty(4 * 256 + 8, dtype=torch.bfloat16, device="cuda")[1:1025].view(4, 256)  # two bytes off the boundary
    with pytest.raises(MoeB200Error):
        ops.rms_norm_quant_fp8(q, s, off, w, 1e-6)


def test_an_error_of_one_call_is_not_reported_by_the_next():
    """A refused allocation (64 TB) leaves the runtime's last error behind; the launches that follow are not to find it."""
    from layered_prefill_b200 import ops
    from layered_prefill_b200._lib import MoeB200Error
    x, w = torch.randn(4, 256).to(torch.bfloat16).cuda(), torch.ones(256, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(x)
    ops.rms_norm(out, x, w, 1e-6)
    want = out.clone()
    with pytest.raises(MoeB200Error):
        ops.allocate_shared_buffer_and_handle(1 << 46)
    ops.rms_norm(out.zero_(), x, w, 1e-6)
    assert torch.equal(out, want)
    with pytest.raises(MoeB200Error):
        ops.allocate_shared_buffer_and_handle(1 << 46)
    assert float((x + x).float().abs().sum()) > 0  # torch checks its launches the same way
