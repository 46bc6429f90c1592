"""Host-side mirror of nanovllm/layers/for_moe/fused_moe.py: `fused_topk`, `moe_align_block_size`,
`fused_experts` / `fused_experts_impl` with the reference's signatures, backed by libmoe_b200.

What is different underneath: one C call runs permutation, both grouped tcgen05 GEMMs (activation
and routed-weight scaling in their epilogues) and the k-slot sum on the current stream; the tile
shape is chosen inside the library from the shapes, so there is no Triton config lookup
(for_moe/fused_moe.py:318-390 has no counterpart here). Quantised paths are rejected, as they are
by the reference's asserts (for_moe/fused_moe.py:248-249,571,607).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops
from ._lib import ACT_CODES, check, lib


def cdiv(a: int, b: int) -> int:
    return -(-a // b)


def fused_topk(hidden_states: torch.Tensor, gating_output: torch.Tensor, topk: int, renormalize: bool):
    """for_moe/fused_moe.py:393-419. Returns (topk_weights f32 [M,k], topk_ids i32 [M,k],
    token_expert_indices i32 [M,k]). bf16 logits are consumed directly (the upcast is exact) and the
    renormalisation is applied by the same kernel."""
    assert hidden_states.shape[0] == gating_output.shape[0], "Number of tokens mismatch"
    M = hidden_states.shape[0]
    dev = hidden_states.device
    topk_weights = torch.empty(M, topk, dtype=torch.float32, device=dev)
    topk_ids = torch.empty(M, topk, dtype=torch.int32, device=dev)
    token_expert_indices = torch.empty(M, topk, dtype=torch.int32, device=dev)
    g = gating_output if gating_output.dtype in (torch.float32, torch.bfloat16) else gating_output.float()
    g = g.contiguous()
    E = g.size(-1)
    with torch.cuda.device(dev):
        check(lib.moe_b200_topk_softmax(g.data_ptr(), int(g.dtype == torch.bfloat16), topk_weights.data_ptr(),
                                        topk_ids.data_ptr(), token_expert_indices.data_ptr(), M, E, topk,
                                        int(bool(renormalize)), torch.cuda.current_stream().cuda_stream))
    return topk_weights, topk_ids, token_expert_indices


def moe_align_block_size(topk_ids: torch.Tensor, block_size: int, num_experts: int
                         ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """for_moe/fused_moe.py:17-70: same buffer sizes and fill value; ids inside an expert come out in
    ascending order (the reference leaves that order to atomic arrival)."""
    max_num_tokens_padded = topk_ids.numel() + num_experts * (block_size - 1)
    sorted_ids = torch.empty((max_num_tokens_padded,), dtype=torch.int32, device=topk_ids.device)
    max_num_m_blocks = cdiv(max_num_tokens_padded, block_size)
    expert_ids = torch.empty((max_num_m_blocks,), dtype=torch.int32, device=topk_ids.device)
    num_tokens_post_pad = torch.empty((1), dtype=torch.int32, device=topk_ids.device)
    ops.moe_align_block_size(topk_ids, num_experts, block_size, sorted_ids, expert_ids, num_tokens_post_pad)
    return sorted_ids, expert_ids, num_tokens_post_pad


class _Workspaces:
    """One scratch tensor per device, reused across calls (no per-call malloc). It grows when a larger request
    comes; outgrown tensors are kept alive, because a CUDA graph captured earlier still holds their address.
    Growing inside a stream capture is refused (the new tensor would belong to the capture's private pool):
    call `reserve_workspace` for the largest batch before capturing. All streams of a device share the buffer,
    so calls on different streams must be ordered by the caller."""

    def __init__(self) -> None:
        self._buf: dict[int, torch.Tensor] = {}
        self._outgrown: list[torch.Tensor] = []

    def get(self, device: torch.device, nbytes: int) -> torch.Tensor:
        idx = device.index if device.index is not None else torch.cuda.current_device()
        cur = self._buf.get(idx)
        if cur is None or cur.numel() < nbytes:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(
                    f"the MoE workspace would have to grow to {nbytes} bytes inside a CUDA-graph capture; "
                    "call fused_moe.reserve_workspace(...) for the largest batch before capturing")
            if cur is not None:
                self._outgrown.append(cur)
            cur = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=torch.device("cuda", idx))
            self._buf[idx] = cur
        return cur


_workspaces = _Workspaces()


def reserve_workspace(device: torch.device, max_tokens: int, num_experts: int, top_k: int, hidden_size: int,
                      intermediate_size_per_partition: int, fp8: bool = False) -> int:
    """Sizes the device's scratch buffer for batches of up to `max_tokens` tokens, so that later calls (inside
    CUDA-graph captures too) never allocate. Returns the size in bytes."""
    args = (int(max_tokens), int(num_experts), int(top_k), int(hidden_size), int(intermediate_size_per_partition))
    nbytes = max(lib.moe_b200_fused_moe_workspace_bytes(*args),
                 lib.moe_b200_fused_experts_fp8_workspace_bytes(*args) if fp8 else 0)
    _workspaces.get(device, nbytes)
    return int(nbytes)


def _check_experts_args(hidden_states, w1, w2, topk_weights, topk_ids, activation, **quant):
    assert hidden_states.size(1) == w1.size(2), f"Hidden size mismatch {hidden_states.size(1)} != {w1.size(2)}"
    assert topk_weights.size() == topk_ids.size(), "topk shape mismatch"
    assert hidden_states.is_contiguous(), "Hidden_states must be contiguous"
    assert w1.stride(-1) == 1, "Stride of last dimension must be 1"
    assert w2.stride(-1) == 1, "Stride of last dimension must be 1"
    if hidden_states.dtype != torch.bfloat16 or w1.dtype != torch.bfloat16 or w2.dtype != torch.bfloat16:
        raise ValueError(f"Unsupported compute_type: {hidden_states.dtype} (this build computes in bfloat16)")
    if activation not in ACT_CODES:
        raise ValueError(f"Unsupported FusedMoe activation: {activation}")
    for name, v in quant.items():
        assert v is None, f"{name} is not supported (the reference asserts the same)"
    if not hidden_states.is_cuda:
        raise RuntimeError("fused_experts needs CUDA tensors; there is no CPU path")
    assert w1.is_contiguous() and w2.is_contiguous(), "expert weights must be contiguous [E, 2I, H] / [E, H, I]"


def fused_experts_impl(hidden_states: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, topk_weights: torch.Tensor,
                       topk_ids: torch.Tensor, inplace: bool = False, activation: str = "silu",
                       apply_router_weight_on_input: bool = False, per_channel_quant: bool = False,
                       global_num_experts: int = -1, expert_map: Optional[torch.Tensor] = None,
                       w1_scale=None, w2_scale=None, w1_zp=None, w2_zp=None, a1_scale=None, a2_scale=None,
                       block_shape=None, w1_bias: Optional[torch.Tensor] = None,
                       w2_bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """for_moe/fused_moe.py:461-633. With e4m3 weights, `w1_scale` / `w2_scale` and `block_shape=[128, 128]` (arguments
    the reference declares and asserts unused) the block-scaled fp8 path runs instead; hidden_states may then be e4m3 with
    `a1_scale` fp32 [T, H / 128] (what ops.rms_norm_quant_fp8 writes). With packed uint8 weights and `block_shape=[0, group]`
    the 4-bit path runs (`w1_scale` / `w2_scale` bf16 per row and group, `w1_zp` / `w2_zp` zero points or None; see quant_w4)."""
    if block_shape is not None and len(block_shape) == 2 and block_shape[0] == 0:
        return _fused_experts_w4(hidden_states, w1, w2, topk_weights, topk_ids, inplace, activation, w1_scale, w2_scale, w1_zp,
                                 w2_zp, block_shape[1], w1_bias, w2_bias, a1_scale, a2_scale, expert_map, global_num_experts,
                                 apply_router_weight_on_input)
    if w1.dtype in (torch.float8_e4m3fn, torch.uint8):
        return _fused_experts_fp8(hidden_states, w1, w2, topk_weights, topk_ids, inplace, activation, w1_scale,
                                  w2_scale, block_shape, w1_bias, w2_bias, a1_scale, a2_scale, w1_zp, w2_zp,
                                  expert_map, apply_router_weight_on_input)
    _check_experts_args(hidden_states, w1, w2, topk_weights, topk_ids, activation, w1_scale=w1_scale,
                        w2_scale=w2_scale, w1_zp=w1_zp, w2_zp=w2_zp, a1_scale=a1_scale, a2_scale=a2_scale,
                        block_shape=block_shape, expert_map=expert_map)
    if apply_router_weight_on_input:
        raise NotImplementedError("apply_router_weight_on_input=True is not used by the reference's models")
    T, H = hidden_states.shape
    E, two_i, _ = w1.shape
    inter = two_i // 2
    assert w2.shape == (E, H, inter), f"w2 shape {tuple(w2.shape)} does not match w13 {tuple(w1.shape)}"
    if global_num_experts not in (-1, E):
        raise NotImplementedError("expert parallelism (global_num_experts != local) is not part of the reference's path")
    k = topk_ids.size(1)
    out = hidden_states if inplace else torch.empty_like(hidden_states)
    if T == 0:
        return out
    tw = topk_weights.to(torch.float32).contiguous()
    ti = topk_ids.to(torch.int32).contiguous()
    dev = hidden_states.device
    nbytes = lib.moe_b200_fused_experts_workspace_bytes(T, E, k, H, inter)
    ws = _workspaces.get(dev, nbytes)
    with torch.cuda.device(dev):
        check(lib.moe_b200_fused_experts(
            hidden_states.data_ptr(), w1.data_ptr(), w2.data_ptr(),
            w1_bias.data_ptr() if w1_bias is not None else 0, w2_bias.data_ptr() if w2_bias is not None else 0,
            tw.data_ptr(), ti.data_ptr(), out.data_ptr(), T, E, k, H, inter, ACT_CODES[activation],
            ws.data_ptr(), ws.numel(), ops.status_word(dev).data_ptr(), torch.cuda.current_stream().cuda_stream))
    return out


def fused_moe_forward_reduce_norm(hidden_states: torch.Tensor, router_logits: torch.Tensor, w13: torch.Tensor,
                                  w2: torch.Tensor, top_k: int, residual: torch.Tensor, norm_weight: torch.Tensor,
                                  eps: float, comm, renormalize: bool = True, activation: str = "silu",
                                  w13_bias: Optional[torch.Tensor] = None, w2_bias: Optional[torch.Tensor] = None):
    """Router + experts + tensor-parallel reduction + the NEXT decoder layer's input_layernorm(hidden, residual)
    (nanovllm/models/qwen3_moe.py:99-116 followed by :262-270) through one library call; the k-slot sum, the
    all-reduce and the add + norm are one kernel for decode-sized batches. residual is updated in place.
    Returns (normed hidden states, residual)."""
    T, H = hidden_states.shape
    E, two_i, _ = w13.shape
    inter = two_i // 2
    assert comm is not None and not comm.disabled and comm.world_size > 1, "needs an initialised CustomAllreduce"
    assert router_logits.shape == (T, E)
    _check_experts_args(hidden_states, w13, w2, router_logits, router_logits, activation)
    assert residual.shape == (T, H) and residual.dtype == torch.bfloat16 and residual.is_contiguous()
    logits = router_logits if router_logits.dtype in (torch.bfloat16, torch.float32) else router_logits.float()
    logits = logits.contiguous()
    normed = torch.empty_like(hidden_states)
    if T == 0:
        return normed, residual
    scratch = torch.empty_like(hidden_states)
    dev = hidden_states.device
    ws = _workspaces.get(dev, lib.moe_b200_fused_moe_workspace_bytes(T, E, top_k, H, inter))
    with torch.cuda.device(dev):
        check(lib.moe_b200_fused_moe_forward_tp_add_rms_norm(
            hidden_states.data_ptr(), logits.data_ptr(), int(logits.dtype == torch.bfloat16), w13.data_ptr(),
            w2.data_ptr(), w13_bias.data_ptr() if w13_bias is not None else 0,
            w2_bias.data_ptr() if w2_bias is not None else 0, residual.data_ptr(), norm_weight.data_ptr(), float(eps),
            normed.data_ptr(), scratch.data_ptr(), T, E, top_k, H, inter, int(bool(renormalize)), ACT_CODES[activation],
            ws.data_ptr(), ws.numel(), comm._ptr, comm.buffer_ptrs[comm.rank], comm.max_size, 0,
            ops.status_word(dev).data_ptr(), torch.cuda.current_stream().cuda_stream))
    return normed, residual


def _fused_experts_fp8(hidden_states, w1, w2, topk_weights, topk_ids, inplace, activation, w1_scale, w2_scale,
                       block_shape, w1_bias, w2_bias, a1_scale, a2_scale, w1_zp, w2_zp, expert_map,
                       apply_router_weight_on_input, out: Optional[torch.Tensor] = None,
                       intermediate_offset: int = 0, intermediate_size: Optional[int] = None, comm=None) -> torch.Tensor:
    """w8a8 e4m3: weights [E, 2I, H] / [E, H, I] with fp32 scales per 128 x 128 block, activations quantised per
    token and 128 columns inside the library (a2_scale stays None), unless they come as e4m3 with a1_scale [T, H / 128]."""
    if not hidden_states.is_cuda:
        raise RuntimeError("fused_experts needs CUDA tensors; there is no CPU path")
    quantized = hidden_states.dtype == torch.float8_e4m3fn
    if hidden_states.dtype != torch.bfloat16 and not quantized:
        raise ValueError(f"Unsupported compute_type: {hidden_states.dtype} (activations enter as bfloat16, or as e4m3 with a1_scale)")
    if quantized and (inplace or comm is not None):
        raise NotImplementedError("e4m3 hidden states cannot take the bf16 result in place, nor go into the fused reduction")
    if w2.dtype != w1.dtype:
        raise ValueError("w1 and w2 must both be e4m3")
    if w1_scale is None or w2_scale is None or block_shape is None or list(block_shape) != [128, 128]:
        raise ValueError("fp8 weights need w1_scale, w2_scale and block_shape=[128, 128]")
    if activation != "silu" or w1_bias is not None or w2_bias is not None:
        raise NotImplementedError("the fp8 path is built for silu without expert biases")
    for name, v in dict(a1_scale=None if quantized else a1_scale, a2_scale=a2_scale, w1_zp=w1_zp, w2_zp=w2_zp,
                        expert_map=expert_map).items():
        assert v is None, f"{name} is not supported"
    if apply_router_weight_on_input:
        raise NotImplementedError("apply_router_weight_on_input=True is not used by the reference's models")
    assert hidden_states.is_contiguous() and w1.is_contiguous() and w2.is_contiguous()
    T, H = hidden_states.shape
    E, two_i, _ = w1.shape
    inter = two_i // 2
    assert w1.shape == (E, 2 * inter, H) and w2.shape == (E, H, inter)
    i_total = inter if intermediate_size is None else int(intermediate_size)
    i_off = int(intermediate_offset)
    if H % 128 or i_total % 128 or inter % 64 or i_off % 64 or i_off < 0 or i_off + inter > i_total:
        raise ValueError(f"fp8 path needs H and I to be multiples of 128 and a rank's slice of I to start and end "
                         f"on multiples of 64 (H={H}, I={i_total}, slice [{i_off}, {i_off + inter}))")
    s1 = w1_scale.to(torch.float32).contiguous()
    s2 = w2_scale.to(torch.float32).contiguous()
    assert s1.shape == (E, 2 * i_total // 128, H // 128), f"w1_scale shape {tuple(s1.shape)}"
    assert s2.shape == (E, H // 128, i_total // 128), f"w2_scale shape {tuple(s2.shape)}"
    k = topk_ids.size(1)
    if quantized and (a1_scale is None or a1_scale.dtype != torch.float32 or a1_scale.shape != (T, H // 128)
                      or not a1_scale.is_contiguous() or a1_scale.device != hidden_states.device):
        raise ValueError(f"e4m3 hidden states need a contiguous a1_scale fp32 [{T}, {H // 128}] on their device")
    if out is None:
        out = hidden_states if inplace else torch.empty_like(hidden_states, dtype=torch.bfloat16)
    assert out.shape == hidden_states.shape and out.dtype == torch.bfloat16 and out.is_contiguous()
    if T == 0:
        return out
    tw = topk_weights.to(torch.float32).contiguous()
    ti = topk_ids.to(torch.int32).contiguous()
    dev = hidden_states.device
    nbytes = lib.moe_b200_fused_experts_fp8_workspace_bytes(T, E, k, H, inter)
    ws = _workspaces.get(dev, nbytes)
    import ctypes
    fptr = ctypes.POINTER(ctypes.c_float)
    with torch.cuda.device(dev):
        if quantized:
            check(lib.moe_b200_fused_experts_fp8_quantized(
                hidden_states.data_ptr(), a1_scale.data_ptr(), w1.data_ptr(), s1.data_ptr(), w2.data_ptr(), s2.data_ptr(),
                tw.data_ptr(), ti.data_ptr(), out.data_ptr(), T, E, k, H, inter, i_off, i_total, ws.data_ptr(), ws.numel(),
                ops.status_word(dev).data_ptr(), torch.cuda.current_stream().cuda_stream))
        elif comm is not None and not comm.disabled and comm.world_size > 1 and T * H * 2 <= comm.max_size:
            check(lib.moe_b200_fused_experts_fp8_tp_reduce(
                hidden_states.data_ptr(), w1.data_ptr(), ctypes.cast(s1.data_ptr(), fptr), w2.data_ptr(),
                ctypes.cast(s2.data_ptr(), fptr), tw.data_ptr(), ti.data_ptr(), out.data_ptr(), T, E, k, H, inter, i_off,
                i_total, ws.data_ptr(), ws.numel(), comm._ptr, comm.buffer_ptrs[comm.rank], comm.max_size, 0,
                ops.status_word(dev).data_ptr(), torch.cuda.current_stream().cuda_stream))
        else:
            check(lib.moe_b200_fused_experts_fp8_tp(
                hidden_states.data_ptr(), w1.data_ptr(), ctypes.cast(s1.data_ptr(), fptr), w2.data_ptr(),
                ctypes.cast(s2.data_ptr(), fptr), tw.data_ptr(), ti.data_ptr(), out.data_ptr(), T, E, k, H, inter, i_off,
                i_total, ws.data_ptr(), ws.numel(), ops.status_word(dev).data_ptr(),
                torch.cuda.current_stream().cuda_stream))
    return out


def _fused_experts_w4(hidden_states, w1, w2, topk_weights, topk_ids, inplace, activation, w1_scale, w2_scale, w1_zp, w2_zp,
                      group_size, w1_bias, w2_bias, a1_scale, a2_scale, expert_map, global_num_experts,
                      apply_router_weight_on_input) -> torch.Tensor:
    """4-bit weights with group scales, bf16 activations: w1 uint8 [E, 2I, H / 2], w2 uint8 [E, H, I / 2] (quant_w4's layout)."""
    if w1.dtype != torch.uint8 or w2.dtype != torch.uint8 or w1.dim() != 3 or w2.dim() != 3:
        raise ValueError("block_shape=[0, group] needs packed uint8 weights [E, 2I, H / 2] and [E, H, I / 2]")
    if w1_scale is None or w2_scale is None or (w1_zp is None) != (w2_zp is None):
        raise ValueError("4-bit weights need w1_scale and w2_scale, and zero points for both or for none")
    if group_size not in (32, 64, 128):
        raise ValueError(f"4-bit weights come in groups of 32, 64 or 128, got {group_size}")
    if activation not in ACT_CODES:
        raise ValueError(f"Unsupported FusedMoe activation: {activation}")
    if a1_scale is not None or a2_scale is not None or expert_map is not None:
        raise ValueError("a1_scale, a2_scale and expert_map are not supported with 4-bit weights")
    if apply_router_weight_on_input or global_num_experts not in (-1, w1.size(0)):
        raise NotImplementedError("apply_router_weight_on_input and expert parallelism are not used by the reference's models")
    if hidden_states.dim() != 2 or topk_ids.dim() != 2 or topk_weights.shape != topk_ids.shape:
        raise ValueError("hidden_states must be [T, H], topk_weights and topk_ids [T, k]")
    T, H = hidden_states.shape
    E, inter, k, g = w1.size(0), w1.size(1) // 2, topk_ids.size(1), group_size
    if H % g or inter % g:
        raise ValueError(f"H and I must be whole numbers of groups of {g} (H={H}, I={inter})")
    tw = topk_weights if topk_weights.dtype is torch.float32 and topk_weights.is_contiguous() else topk_weights.float().contiguous()
    ti = topk_ids if topk_ids.dtype is torch.int32 and topk_ids.is_contiguous() else topk_ids.to(torch.int32).contiguous()
    bf16, u8, dev = torch.bfloat16, torch.uint8, hidden_states.device
    ops._check("fused_experts (4-bit)", dev, "hidden_states w1 w2 w1_scale w2_scale w1_zp w2_zp w1_bias w2_bias topk_weights topk_ids",
               (hidden_states, bf16, (T, H)), (w1, u8, (E, 2 * inter, H // 2)), (w2, u8, (E, H, inter // 2)),
               (w1_scale, bf16, (E, 2 * inter, H // g)), (w2_scale, bf16, (E, H, inter // g)), (w1_zp, u8, (E, 2 * inter, H // g)),
               (w2_zp, u8, (E, H, inter // g)), (w1_bias, bf16, (E, 2 * inter)), (w2_bias, bf16, (E, H)),
               (tw, torch.float32, (T, k)), (ti, torch.int32, (T, k)))
    out = hidden_states if inplace else torch.empty_like(hidden_states)
    nbytes = lib.moe_b200_fused_experts_w4_workspace_bytes(T, E, k, H, inter)
    # not the shared scratch buffer: a tensor of the current stream (or of the capture's own pool), a few KB a slot
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    p = ops._ptr
    ops._launch(lib.moe_b200_fused_experts_w4, dev, p(hidden_states), p(w1), p(w1_scale), p(w1_zp), p(w1_bias), p(w2), p(w2_scale),
                p(w2_zp), p(w2_bias), p(tw), p(ti), p(out), T, E, k, H, inter, g, ACT_CODES[activation], p(ws), nbytes)
    return out


def quant_w4(weight: torch.Tensor, group_size: int = 128, zero_points: bool = False):
    """Rounds weights [..., N, K] to 4-bit codes with a bf16 scale (and, with zero_points, a zero point) per row and group of
    group_size columns: weight ~ (code - zero) * scale, zero = 8 without zero points. Returns (codes uint8 [..., N, K / 2], two a
    byte with the even column in the low nibble, scales bf16 [..., N, K / group_size], zeros uint8 or None). Done once when
    weights are loaded; works on any device."""
    if group_size not in (32, 64, 128) or weight.size(-1) % group_size:
        raise ValueError(f"group_size must be 32, 64 or 128 and divide the {weight.size(-1)} columns")
    w = weight.float().unflatten(-1, (-1, group_size))
    if zero_points:
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scale = ((hi - lo) / 15).to(torch.bfloat16)
        s = scale.float()
        zero = torch.where(s > 0, (-lo / s).round(), torch.zeros_like(s)).clamp(0, 15)
    else:
        scale = (w.abs().amax(-1) / 7.5).to(torch.bfloat16)
        s, zero = scale.float(), torch.full_like(scale, 8, dtype=torch.float32)
    code = torch.where(s[..., None] > 0, w / s[..., None], torch.zeros_like(w)).add_(zero[..., None]).round_().clamp_(0, 15)
    code = code.to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale, zero.to(torch.uint8) if zero_points else None


def shard_w4_expert_weights(w13, w2, tp_rank: int, tp_size: int, group_size: int, activation: str = "silu"):
    """Slices 4-bit expert weights over the intermediate dimension the way FusedMoE.weight_loader slices bf16 ones
    (nanovllm/layers/fused_moe.py:400-470): for silu, whose w13 holds the gate rows and then the up rows, this rank's part of
    each; for swigluoai, whose gate and up rows alternate, the rows between. w13 and w2 are quant_w4's (codes, scales, zeros) of
    [E, 2I, H] and [E, H, I]; a rank's share of I has to be a whole number of groups. Returns the two triples of this rank. Works
    on any device."""
    if activation not in ACT_CODES:
        raise ValueError(f"Unsupported FusedMoe activation: {activation}")
    inter = w13[0].size(1) // 2
    if inter % tp_size or (inter // tp_size) % group_size:
        raise ValueError(f"a rank's share of I={inter} over {tp_size} ranks must be a whole number of groups of {group_size}")
    ip = inter // tp_size
    lo, hi = tp_rank * ip, (tp_rank + 1) * ip

    def rows(t):
        if t is None:
            return None
        if activation == "swigluoai":
            return t[:, 2 * lo:2 * hi].contiguous()
        return torch.cat([t[:, lo:hi], t[:, inter + lo:inter + hi]], dim=1)

    cols = lambda t, per: None if t is None else t[:, :, lo // per:hi // per].contiguous()  # noqa: E731
    return tuple(rows(t) for t in w13), tuple(cols(t, per) for t, per in zip(w2, (2, group_size, group_size)))


def shard_fp8_expert_weights(w13_q: torch.Tensor, w2_q: torch.Tensor, tp_rank: int, tp_size: int):
    """Slices e4m3 expert weights over the intermediate dimension the way FusedMoE.weight_loader slices bf16 ones
    (nanovllm/layers/fused_moe.py:400-470): w13 [E, 2I, H] -> its gate rows then its up rows of this rank, w2 [E, H, I] ->
    its columns. Returns (w13_local, w2_local, intermediate_offset); the scales are NOT sliced (the kernels index the
    unsharded scale tensors by global position). Works on any device."""
    E, two_i, _ = w13_q.shape
    inter = two_i // 2
    if inter % tp_size:
        raise ValueError(f"intermediate size {inter} is not divisible by the tensor-parallel size {tp_size}")
    ip = inter // tp_size
    lo, hi = tp_rank * ip, (tp_rank + 1) * ip
    b13, b2 = w13_q.view(torch.uint8), w2_q.view(torch.uint8)
    w13_local = torch.cat([b13[:, lo:hi], b13[:, inter + lo:inter + hi]], dim=1).contiguous().view(w13_q.dtype)
    w2_local = b2[:, :, lo:hi].contiguous().view(w2_q.dtype)
    return w13_local, w2_local, lo


def fused_experts_fp8_shard(hidden_states: torch.Tensor, w13_q: torch.Tensor, w13_scale: torch.Tensor,
                            w2_q: torch.Tensor, w2_scale: torch.Tensor, topk_weights: torch.Tensor,
                            topk_ids: torch.Tensor, intermediate_offset: int, intermediate_size: int,
                            out: Optional[torch.Tensor] = None, comm=None) -> torch.Tensor:
    """One tensor-parallel rank of the fp8 experts: w13_q [E, 2*Ip, H] / w2_q [E, H, Ip] hold the slice
    [intermediate_offset, intermediate_offset + Ip) of the intermediate dimension (sharded as FusedMoE.weight_loader
    shards bf16 weights), the scales are those of the unsharded weights. Returns this rank's partial sum, or, with
    `comm` (an initialised CustomAllreduce), the layer's output: the k-slot sum then runs inside the all-reduce."""
    return _fused_experts_fp8(hidden_states, w13_q, w2_q, topk_weights, topk_ids, False, "silu", w13_scale, w2_scale,
                              [128, 128], None, None, None, None, None, None, None, False, out=out,
                              intermediate_offset=intermediate_offset, intermediate_size=intermediate_size, comm=comm)


def pre_moe(hidden_states: torch.Tensor, residual: torch.Tensor, norm_weight: torch.Tensor, eps: float,
            gate_weight: torch.Tensor, top_k: int, renormalize: bool = True, return_logits: bool = False):
    """The decoder layer's steps in front of the MoE block (nanovllm/models/qwen3_moe.py:276-282 and :100-110):
    post_attention_layernorm(hidden_states, residual) -> gate -> softmax/top-k, one library call.

    hidden_states: bf16 [T, H] attention output (not modified); residual: bf16 [T, H], updated in place;
    norm_weight: RMSNorm.weight [H]; gate_weight: ReplicatedLinear.weight [E, H].
    Returns (normed hidden states, residual, topk_weights fp32 [T, k], topk_ids int32 [T, k][, router_logits bf16 [T, E]])."""
    if not hidden_states.is_cuda:
        raise RuntimeError("pre_moe needs CUDA tensors; there is no CPU path")
    for t in (hidden_states, residual, norm_weight, gate_weight):
        assert t.dtype == torch.bfloat16 and t.is_contiguous()
    T, H = hidden_states.shape
    E = gate_weight.size(0)
    assert residual.shape == (T, H) and norm_weight.numel() == H and gate_weight.shape == (E, H)
    dev = hidden_states.device
    normed = torch.empty_like(hidden_states)
    tw = torch.empty(T, top_k, dtype=torch.float32, device=dev)
    ti = torch.empty(T, top_k, dtype=torch.int32, device=dev)
    logits = torch.empty(T, E, dtype=torch.bfloat16, device=dev) if return_logits else None
    if T > 0:
        nbytes = lib.moe_b200_pre_moe_workspace_bytes(T, H, E)
        ws = _workspaces.get(dev, nbytes)
        with torch.cuda.device(dev):
            check(lib.moe_b200_add_rms_norm_router(
                hidden_states.data_ptr(), residual.data_ptr(), norm_weight.data_ptr(), float(eps), gate_weight.data_ptr(),
                normed.data_ptr(), logits.data_ptr() if logits is not None else 0, tw.data_ptr(), ti.data_ptr(), T, H, E,
                top_k, 1 if renormalize else 0, ws.data_ptr(), ws.numel(), ops.status_word(dev).data_ptr(),
                torch.cuda.current_stream().cuda_stream))
    return (normed, residual, tw, ti, logits) if return_logits else (normed, residual, tw, ti)


def fused_moe_forward_fp8(hidden_states: torch.Tensor, router_logits: torch.Tensor, w13_q: torch.Tensor,
                          w13_scale: torch.Tensor, w2_q: torch.Tensor, w2_scale: torch.Tensor, top_k: int,
                          renormalize: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Router + fp8 experts: what FusedMoE.forward does (layers/fused_moe.py:590-612) with e4m3 block-scaled weights."""
    tw, ti, _ = fused_topk(hidden_states, router_logits, top_k, renormalize)
    return _fused_experts_fp8(hidden_states, w13_q, w2_q, tw, ti, False, "silu", w13_scale, w2_scale, [128, 128], None,
                              None, None, None, None, None, None, False, out=out)


def fused_moe_forward_w4(hidden_states: torch.Tensor, router_logits: torch.Tensor, w13, w2, top_k: int, group_size: int,
                         renormalize: bool = True, activation: str = "silu", inplace: bool = False) -> torch.Tensor:
    """Router + 4-bit experts: what FusedMoE.forward does (layers/fused_moe.py:590-612) with quant_w4's (codes, scales, zeros)
    of w13 [E, 2I, H] and w2 [E, H, I]."""
    tw, ti, _ = fused_topk(hidden_states, router_logits, top_k, renormalize)
    return fused_experts_impl(hidden_states, w13[0], w2[0], tw, ti, inplace, activation, w1_scale=w13[1], w2_scale=w2[1],
                              w1_zp=w13[2], w2_zp=w2[2], block_shape=[0, group_size])


class _TopkWithLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gating_output, topk, renormalize, token_mask):
        T, E = gating_output.shape
        dev = gating_output.device
        tw = torch.empty(T, topk, dtype=torch.float32, device=dev)
        ti = torch.empty(T, topk, dtype=torch.int32, device=dev)
        losses = torch.empty(2, dtype=torch.float32, device=dev)
        counts = torch.empty(E, dtype=torch.int32, device=dev)
        num = torch.empty(1, dtype=torch.int32, device=dev)
        mean_probs = torch.empty(E, dtype=torch.float32, device=dev)
        if T > 0:
            ops.topk_softmax_renorm(tw, ti, gating_output, renormalize)
        ops.router_loss(losses, counts, num, mean_probs, gating_output, ti, token_mask)
        ctx.save_for_backward(gating_output, ti, counts, num, token_mask)
        ctx.renormalize = renormalize
        ctx.mark_non_differentiable(ti, counts)
        ctx.set_materialize_grads(False)
        return tw, ti, losses, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_tw, _g_ti, g_losses, _g_counts):
        gating_output, ti, counts, num, token_mask = ctx.saved_tensors
        if g_tw is None and g_losses is None:
            return None, None, None, None
        grad = torch.empty_like(gating_output)
        ops.router_backward(grad, gating_output, ti, counts, num, None if g_losses is None else g_losses.contiguous(),
                            None if g_tw is None else g_tw.contiguous(), ctx.renormalize, token_mask)
        return grad, None, None, None


def fused_topk_with_loss(gating_output: torch.Tensor, topk: int, renormalize: bool, token_mask: Optional[torch.Tensor] = None):
    """`fused_topk` for training a router: returns (topk_weights fp32 [T, k], topk_ids int32 [T, k], balance_loss, z_loss,
    counts int32 [E]). topk_weights and the losses (see ops.router_loss) are differentiable once with respect to
    gating_output (fp32 or bf16 [T, E]); tokens that token_mask (bool [T]) leaves out do not count and get no gradient,
    not through their routed weights either. Balanced routing has a balance loss of k. Weight the losses by their
    coefficients and add them to the task's loss. A captured backward pass needs what torch asks for: a graph of its own, built
    in the capture, whose leaves no eager graph holds."""
    if gating_output.dim() != 2 or gating_output.dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError("fused_topk_with_loss: gating_output must be float32 or bfloat16 [T, E]")
    if not gating_output.is_cuda:
        raise RuntimeError("fused_topk_with_loss needs CUDA tensors; there is no CPU path")
    if not 0 < topk <= gating_output.size(1):
        raise RuntimeError(f"fused_topk_with_loss: need 0 < topk <= {gating_output.size(1)}, got {topk}")
    tw, ti, losses, counts = _TopkWithLoss.apply(gating_output.contiguous(), int(topk), bool(renormalize), token_mask)
    return tw, ti, losses[0], losses[1], counts


def per_token_group_quant_fp8(x: torch.Tensor, group_size: int = 128):
    """x bf16 [rows, cols] -> (e4m3 [rows, cols], fp32 scales [rows, cols / 128]); the quantisation the fp8 path
    applies to its activations."""
    if group_size != 128:
        raise ValueError("group_size must be 128")
    if not x.is_cuda:
        raise RuntimeError("per_token_group_quant_fp8 needs a CUDA tensor; there is no CPU path")
    assert x.dtype == torch.bfloat16 and x.dim() == 2 and x.is_contiguous() and x.size(1) % 128 == 0
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    s = torch.empty((x.size(0), x.size(1) // 128), dtype=torch.float32, device=x.device)
    import ctypes
    with torch.cuda.device(x.device):
        check(lib.moe_b200_quant_fp8_per_token_group(
            x.data_ptr(), x.size(0), x.size(1), q.data_ptr(), ctypes.cast(s.data_ptr(), ctypes.POINTER(ctypes.c_float)),
            torch.cuda.current_stream().cuda_stream))
    return q, s


def fused_experts(hidden_states: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, w1_bias: Optional[torch.Tensor],
                  w2_bias: Optional[torch.Tensor], topk_weights: torch.Tensor, topk_ids: torch.Tensor,
                  inplace: bool = False, activation: str = "silu", apply_router_weight_on_input: bool = False,
                  per_channel_quant: bool = False, global_num_experts: int = -1,
                  expert_map: Optional[torch.Tensor] = None, w1_scale=None, w2_scale=None, w1_zp=None, w2_zp=None,
                  a1_scale=None, a2_scale=None, block_shape=None, allow_deep_gemm: bool = False) -> torch.Tensor:
    """for_moe/fused_moe.py:422-460."""
    return fused_experts_impl(hidden_states, w1, w2, topk_weights, topk_ids, inplace, activation,
                              apply_router_weight_on_input, per_channel_quant, global_num_experts, expert_map,
                              w1_scale, w2_scale, w1_zp, w2_zp, a1_scale, a2_scale, block_shape, w1_bias, w2_bias)


def fused_moe_forward(hidden_states: torch.Tensor, router_logits: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor,
                      top_k: int, renormalize: bool = True, activation: str = "silu", inplace: bool = True,
                      w13_bias: Optional[torch.Tensor] = None, w2_bias: Optional[torch.Tensor] = None,
                      comm=None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Router + experts (+ tensor-parallel reduction when `comm` is an initialised CustomAllreduce) through
    one library call: what FusedMoE.forward followed by maybe_all_reduce_tensor_model_parallel does
    (nanovllm/layers/fused_moe.py:746-787, nanovllm/models/qwen3_moe.py:99-116). `out` (bf16 [T, H]) is used
    as the destination when given; otherwise the result overwrites hidden_states (inplace) or a new tensor."""
    T, H = hidden_states.shape
    E, two_i, _ = w13.shape
    inter = two_i // 2
    assert router_logits.shape == (T, E), "router_logits must be [tokens, experts]"
    _check_experts_args(hidden_states, w13, w2, router_logits, router_logits, activation)
    logits = router_logits if router_logits.dtype in (torch.bfloat16, torch.float32) else router_logits.float()
    logits = logits.contiguous()
    if out is None:
        out = hidden_states if inplace else torch.empty_like(hidden_states)
    else:
        assert out.shape == hidden_states.shape and out.dtype == hidden_states.dtype and out.is_contiguous()
    if T == 0:
        return out
    dev = hidden_states.device
    nbytes = lib.moe_b200_fused_moe_workspace_bytes(T, E, top_k, H, inter)
    ws = _workspaces.get(dev, nbytes)
    stream = torch.cuda.current_stream().cuda_stream
    b13 = w13_bias.data_ptr() if w13_bias is not None else 0
    b2 = w2_bias.data_ptr() if w2_bias is not None else 0
    with torch.cuda.device(dev):
        if comm is not None and not comm.disabled and comm.world_size > 1:
            check(lib.moe_b200_fused_moe_forward_tp(
                hidden_states.data_ptr(), logits.data_ptr(), int(logits.dtype == torch.bfloat16), w13.data_ptr(),
                w2.data_ptr(), b13, b2, out.data_ptr(), T, E, top_k, H, inter, int(bool(renormalize)),
                ACT_CODES[activation], ws.data_ptr(), ws.numel(), comm._ptr, comm.buffer_ptrs[comm.rank],
                comm.max_size, 0, ops.status_word(dev).data_ptr(), stream))
        else:
            check(lib.moe_b200_fused_moe_forward(
                hidden_states.data_ptr(), logits.data_ptr(), int(logits.dtype == torch.bfloat16), w13.data_ptr(),
                w2.data_ptr(), b13, b2, out.data_ptr(), 0, 0, T, E, top_k, H, inter, int(bool(renormalize)),
                ACT_CODES[activation], ws.data_ptr(), ws.numel(), ops.status_word(dev).data_ptr(), stream))
    return out
