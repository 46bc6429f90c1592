"""Host-side mirror of the hot-path functions of the reference's `nanovllm.ops` extension
(csrc/ops.cpp:97-159): same names, same argument order, torch tensors in, results written in place.
Each function forwards raw pointers to libmoe_b200 on the current CUDA stream; there is no
fallback -- a CPU tensor or a missing library is an error.
"""
from __future__ import annotations

import ctypes
from typing import List, Tuple

import torch

from . import _lib
from ._lib import check, lib


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _need_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("libmoe_b200 ops take CUDA tensors only (there is no CPU path)")


_status_words: dict[int, torch.Tensor] = {}


def status_word(device: torch.device) -> torch.Tensor:
    """One zero-initialised int32 per device; kernels store a code there when a bounded wait runs out."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _status_words:
        _status_words[idx] = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
    return _status_words[idx]


def launch_count() -> int:
    """Kernels this library has launched in this process so far (graph replays are not seen)."""
    return int(lib.moe_b200_launch_count())


def read_status(device: torch.device | None = None) -> int:
    """Synchronise the current stream and return the device status word (0 = no device-side timeout)."""
    dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
    v = ctypes.c_int32(0)
    with torch.cuda.device(dev):
        check(lib.moe_b200_read_status(status_word(dev).data_ptr(), ctypes.byref(v), _stream()))
    return int(v.value)


def _norm_args(out: torch.Tensor, input: torch.Tensor, weight: torch.Tensor):  # noqa: A002
    _need_cuda(out, input, weight)
    if input.dtype != torch.bfloat16 or out.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise RuntimeError("rms_norm: bfloat16 tensors only")
    assert input.is_contiguous() and out.is_contiguous() and weight.is_contiguous() and out.shape == input.shape
    H = input.size(-1)
    assert weight.numel() == H
    return (input.numel() // H if H else 0), H


def rms_norm(out: torch.Tensor, input: torch.Tensor, weight: torch.Tensor, epsilon: float) -> None:  # noqa: A002
    """csrc/ops.cpp:16-21. out = bf16(bf16(x * rsqrt(mean(x^2) + eps)) * weight); out may be input."""
    T, H = _norm_args(out, input, weight)
    with torch.cuda.device(input.device):
        check(lib.moe_b200_rms_norm(out.data_ptr(), input.data_ptr(), weight.data_ptr(), float(epsilon), T, H, _stream()))


def add_rms_norm(out: torch.Tensor, residual: torch.Tensor, input: torch.Tensor, weight: torch.Tensor,  # noqa: A002
                 epsilon: float) -> None:
    """csrc/ops.cpp:22-27. residual <- bf16(input + residual) in place, out = its RMS norm times weight."""
    T, H = _norm_args(out, input, weight)
    _need_cuda(residual)
    assert residual.dtype == torch.bfloat16 and residual.is_contiguous() and residual.shape == input.shape
    with torch.cuda.device(input.device):
        check(lib.moe_b200_add_rms_norm(out.data_ptr(), residual.data_ptr(), input.data_ptr(), weight.data_ptr(),
                                        float(epsilon), T, H, _stream()))


def topk_softmax(topk_weights: torch.Tensor, topk_indices: torch.Tensor, token_expert_indices: torch.Tensor,
                 gating_output: torch.Tensor) -> None:
    """csrc/ops.cpp:46-51. gating_output fp32 (or bf16) [T, E]; outputs [T, k]."""
    _need_cuda(topk_weights, topk_indices, token_expert_indices, gating_output)
    assert gating_output.is_contiguous() and topk_weights.is_contiguous() and topk_indices.is_contiguous()
    assert topk_weights.dtype == torch.float32 and topk_indices.dtype == torch.int32
    if gating_output.dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError("topk_softmax: gating_output must be float32 or bfloat16")
    E = gating_output.size(-1)
    T = gating_output.numel() // E if E else 0
    k = topk_weights.size(-1)
    tei = 0
    if token_expert_indices is not None:
        assert token_expert_indices.dtype == torch.int32 and token_expert_indices.is_contiguous()
        tei = token_expert_indices.data_ptr()
    with torch.cuda.device(gating_output.device):
        check(lib.moe_b200_topk_softmax(gating_output.data_ptr(), int(gating_output.dtype == torch.bfloat16),
                                        topk_weights.data_ptr(), topk_indices.data_ptr(), tei, T, E, k, 0, _stream()))


def topk_softmax_renorm(topk_weights: torch.Tensor, topk_indices: torch.Tensor, gating_output: torch.Tensor,
                        renormalize: bool) -> None:
    """topk_softmax with the renormalisation of fused_topk folded in (one launch, bf16 or fp32 logits)."""
    _need_cuda(topk_weights, topk_indices, gating_output)
    assert gating_output.is_contiguous() and topk_weights.is_contiguous() and topk_indices.is_contiguous()
    E = gating_output.size(-1)
    T = gating_output.numel() // E if E else 0
    with torch.cuda.device(gating_output.device):
        check(lib.moe_b200_topk_softmax(gating_output.data_ptr(), int(gating_output.dtype == torch.bfloat16),
                                        topk_weights.data_ptr(), topk_indices.data_ptr(), 0, T, E,
                                        topk_weights.size(-1), int(bool(renormalize)), _stream()))


# ---------------------------------------------------------------- low-precision operators around the block, router losses
_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream(device).cuda_stream, without the Stream object (5 us a call)


_MAX_ROWS = 2**30 - 1  # tokens of a call: their number crosses the C interface as an int
# Below these the library asks for no workspace, and asking it is saved; its own numbers are kOneCta, kOneCtaLogits (router_loss.cu)
# and kPreparedChunks (w4_gemv.cu), and a test compares the two.
_LOSS_ALONE_TOKENS, _LOSS_ALONE_LOGITS = 128, 16384
_W4_SMALL = 8192


def _launch(fn, device: torch.device, *args) -> None:
    """check(fn(*args, current stream)) with `device` current."""
    idx = device.index
    if idx == torch._C._cuda_getDevice():
        status = fn(*args, _raw_stream(idx))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(idx))
    if status != 0:
        check(status)


def _check(op: str, device: torch.device, names: str, *specs) -> None:
    """specs, named by names: (tensor or None, dtype, shape); contiguous tensors of that CUDA device, dtype and shape."""
    idx = device.index
    for t, dtype, shape in specs:
        if t is not None and (t.get_device() != idx or t.dtype is not dtype or t.shape != shape or not t.is_contiguous()):
            break
    else:
        if device.type == "cuda":
            return
    if device.type != "cuda":
        raise RuntimeError(f"{op}: takes CUDA tensors only (got one on {device}); there is no CPU path")
    for name, (t, dtype, shape) in zip(names.split(), specs):
        if t is None:
            continue
        if t.device != device:
            raise RuntimeError(f"{op}: {name} must be on {device} like the other tensors, got {t.device}")
        if t.dtype != dtype:
            raise RuntimeError(f"{op}: {name} must be {dtype}, got {t.dtype}")
        if t.shape != shape:
            raise RuntimeError(f"{op}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
        if not t.is_contiguous():
            raise RuntimeError(f"{op}: {name} must be contiguous")


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _norm_quant(op, out, scales, residual, input, weight, epsilon, group_size, normed_out, residual_out):  # noqa: A002
    bf16, shape, device = torch.bfloat16, input.shape, input.device
    H = shape[-1] if shape else 0
    T = input.numel() // H if H else 0
    if T > _MAX_ROWS:
        raise RuntimeError(f"{op}: at most {_MAX_ROWS} tokens, got {T}")
    groups = 1 if group_size == -1 or (group_size == H and H != 128) else H // 128
    _check(op, device, "input out weight scales residual residual_out normed_out", (input, bf16, shape),
           (out, torch.float8_e4m3fn, shape), (weight, bf16, (H,)), (scales, torch.float32, (*shape[:-1], groups)),
           (residual, bf16, shape), (residual_out, bf16, shape), (normed_out, bf16, shape))
    _launch(lib.moe_b200_rms_norm_quant_fp8, device, out.data_ptr(), scales.data_ptr(), _ptr(normed_out),
            _ptr(residual_out), _ptr(residual), input.data_ptr(), weight.data_ptr(), epsilon, T, H, group_size)


def rms_norm_quant_fp8(out: torch.Tensor, scales: torch.Tensor, input: torch.Tensor, weight: torch.Tensor,  # noqa: A002
                       epsilon: float, group_size: int = 128, normed_out: torch.Tensor | None = None) -> None:
    """RMS norm with an e4m3 output: y = input * rsqrt(mean(input^2) + eps) * weight in fp32, scales = max(|y|, 1e-10) / 448 over
    each group of 128 columns ([.., H / 128]) or, with group_size -1, over each token ([.., 1]), out = e4m3(y / scale).
    normed_out, if given, gets bf16(y), rounded once (`rms_norm` also rounds before the weight). The pair (out, scales) with groups
    of 128 is what `fused_experts` takes as hidden states and `a1_scale` next to e4m3 weights."""
    _norm_quant("rms_norm_quant_fp8", out, scales, None, input, weight, epsilon, group_size, normed_out, None)


def add_rms_norm_quant_fp8(out: torch.Tensor, scales: torch.Tensor, residual: torch.Tensor, input: torch.Tensor,  # noqa: A002
                           weight: torch.Tensor, epsilon: float, group_size: int = 128,
                           normed_out: torch.Tensor | None = None, residual_out: torch.Tensor | None = None) -> None:
    """`rms_norm_quant_fp8` of residual <- bf16(input + residual): the sum is written to residual_out, or to residual itself."""
    _norm_quant("add_rms_norm_quant_fp8", out, scales, residual, input, weight, epsilon, group_size, normed_out,
                residual if residual_out is None else residual_out)


def w4_linear(out: torch.Tensor, input: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor,  # noqa: A002
              zeros: torch.Tensor | None = None, bias: torch.Tensor | None = None) -> None:
    """out[.., N] = input[.., K] @ W^T + bias for 4-bit weights W[n, k] = (code - zero) * scale, built for few tokens (any number
    works). qweight uint8 [N, K / 2], two codes a byte, the low nibble is the even k; scales bf16 [N, K / group], groups of 32, 64 or
    128; zeros uint8 0..15 like scales (8 without it); bias bf16 [N]. A two-dimensional input may have rows further than K apart
    (a multiple of 8 elements); out must not share memory with it. The activations enter the products as 16-bit integers times a
    power of two for every 128 columns: exact down to 2^-7 of their largest, off by at most 2^-15 of it below; where a few columns stand
    out so far that this would show in rows without a weight for them (one of 100 times the rest, say), 16 bits more are taken. Sums
    are fp32. `fused_moe.quant_w4` makes such weights."""
    shape, q_shape, s_shape = input.shape, qweight.shape, scales.shape
    if len(q_shape) != 2 or len(s_shape) != 2 or not shape or not shape[-1] or not q_shape[0] or not s_shape[1]:
        raise RuntimeError("w4_linear: qweight must be [N, K / 2], scales [N, K / group] and input [.., K]")
    K, N, groups = shape[-1], q_shape[0], s_shape[1]
    M = input.numel() // K
    if M > _MAX_ROWS:
        raise RuntimeError(f"w4_linear: at most {_MAX_ROWS} tokens, got {M}")
    bf16, u8, device, ld, checked = torch.bfloat16, torch.uint8, qweight.device, K, (input, torch.bfloat16, shape)
    if len(shape) == 2 and not input.is_contiguous() and input.stride(1) == 1:
        ld, checked = input.stride(0), (input[:1], bf16, (min(M, 1), K))
    _check("w4_linear", device, "input out qweight scales zeros bias", checked, (out, bf16, (*shape[:-1], N)),
           (qweight, u8, (N, K // 2)), (scales, bf16, (N, groups)), (zeros, u8, (N, groups)), (bias, bf16, (N,)))
    group = K // groups if K % groups == 0 else -1
    ws, nbytes = None, 0
    if M * (K + 127) > _W4_SMALL:
        nbytes = lib.moe_b200_w4_linear_workspace_bytes(M, K, group)
        ws = torch.empty(nbytes, dtype=u8, device=device) if nbytes else None
    _launch(lib.moe_b200_w4_linear, device, out.data_ptr(), input.data_ptr(), ld, qweight.data_ptr(), scales.data_ptr(),
            zeros.data_ptr() if zeros is not None else 0, bias.data_ptr() if bias is not None else 0, M, N, K, group,
            ws.data_ptr() if ws is not None else 0, nbytes)


def _router_args(op, gating_output, topk_ids, token_mask):
    if gating_output.dim() != 2 or topk_ids.dim() != 2:
        raise RuntimeError(f"{op}: gating_output must be [T, E] and topk_ids [T, k]")
    if gating_output.dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError(f"{op}: gating_output must be float32 or bfloat16")
    T, E = gating_output.shape
    k = topk_ids.size(1)
    if T > _MAX_ROWS:
        raise RuntimeError(f"{op}: at most {_MAX_ROWS} tokens, got {T}")
    specs = ((gating_output, gating_output.dtype, (T, E)), (topk_ids, torch.int32, (T, k)),
             (token_mask, torch.uint8 if token_mask is not None and token_mask.dtype == torch.uint8 else torch.bool, (T,)))
    return T, E, k, specs


def router_loss(losses: torch.Tensor, counts: torch.Tensor, num_tokens: torch.Tensor, mean_probs: torch.Tensor,
                gating_output: torch.Tensor, topk_ids: torch.Tensor, token_mask: torch.Tensor | None = None) -> None:
    """Balance loss, z loss and per-expert counts of a routed batch. gating_output fp32 or bf16 [T, E], topk_ids int32 [T, k] (ids
    outside [0, E) are not counted), token_mask bool [T] (False: padding, neither read nor counted). With n counted tokens
    (divisions by at least 1) and p = softmax(gating_output): counts int32 [E], num_tokens int32 [1] = n, mean_probs fp32 [E] =
    sum p / n, losses fp32 [2] = (E * sum(counts / n * mean_probs), sum logsumexp^2 / n). E <= 1024. Same bits on every run."""
    T, E, k, specs = _router_args("router_loss", gating_output, topk_ids, token_mask)
    dev = gating_output.device
    _check("router_loss", dev, "gating_output topk_ids token_mask losses counts num_tokens mean_probs", *specs,
           (losses, torch.float32, (2,)), (counts, torch.int32, (E,)), (num_tokens, torch.int32, (1,)),
           (mean_probs, torch.float32, (E,)))
    ws, nbytes = None, 0
    if T > _LOSS_ALONE_TOKENS or T * E > _LOSS_ALONE_LOGITS:
        nbytes = lib.moe_b200_router_loss_workspace_bytes(T, E)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _launch(lib.moe_b200_router_loss, dev, losses.data_ptr(), counts.data_ptr(), num_tokens.data_ptr(), mean_probs.data_ptr(),
            gating_output.data_ptr(), gating_output.dtype == torch.bfloat16, topk_ids.data_ptr(), _ptr(token_mask), T, E, k,
            _ptr(ws), nbytes)


def router_backward(grad_logits: torch.Tensor, gating_output: torch.Tensor, topk_ids: torch.Tensor, counts: torch.Tensor,
                    num_tokens: torch.Tensor, grad_losses: torch.Tensor | None, grad_topk_weights: torch.Tensor | None,
                    renormalize: bool, token_mask: torch.Tensor | None = None) -> None:
    """grad_logits (like gating_output) = gradient of grad_losses . (balance, z) + sum(grad_topk_weights * topk_weights) with respect
    to gating_output; counts and num_tokens come from `router_loss` (summed over the ranks of a data-parallel job), the routed weights
    are those of `topk_softmax` / `topk_softmax_renorm`. grad_losses fp32 [2] and grad_topk_weights fp32 [T, k] may be None. Rows that
    token_mask leaves out are zero. grad_logits must not share memory with gating_output."""
    T, E, k, specs = _router_args("router_backward", gating_output, topk_ids, token_mask)
    dev = gating_output.device
    _check("router_backward", dev, "gating_output topk_ids token_mask grad_logits counts num_tokens grad_losses grad_topk_weights",
           *specs, (grad_logits, gating_output.dtype, (T, E)), (counts, torch.int32, (E,)), (num_tokens, torch.int32, (1,)),
           (grad_losses, torch.float32, (2,)), (grad_topk_weights, torch.float32, (T, k)))
    _launch(lib.moe_b200_router_backward, dev, grad_logits.data_ptr(), gating_output.data_ptr(),
            gating_output.dtype == torch.bfloat16, topk_ids.data_ptr(), _ptr(counts), _ptr(num_tokens), _ptr(grad_losses),
            _ptr(grad_topk_weights), _ptr(token_mask), T, E, k, bool(renormalize))


def moe_align_block_size(topk_ids: torch.Tensor, num_experts: int, block_size: int, sorted_token_ids: torch.Tensor,
                         experts_ids: torch.Tensor, num_tokens_post_pad: torch.Tensor) -> None:
    """csrc/ops.cpp:53-60."""
    _need_cuda(topk_ids, sorted_token_ids, experts_ids, num_tokens_post_pad)
    if topk_ids.dtype != torch.int32:
        raise RuntimeError("moe_align_block_size: topk_ids must be int32")
    assert topk_ids.is_contiguous() and sorted_token_ids.is_contiguous() and experts_ids.is_contiguous()
    numel = topk_ids.numel()
    ws_bytes = lib.moe_b200_align_workspace_bytes(numel, num_experts)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=topk_ids.device)
    with torch.cuda.device(topk_ids.device):
        check(lib.moe_b200_moe_align_block_size(topk_ids.data_ptr(), numel, num_experts, block_size,
                                                sorted_token_ids.data_ptr(), sorted_token_ids.numel(),
                                                experts_ids.data_ptr(), experts_ids.numel(),
                                                num_tokens_post_pad.data_ptr(), ws.data_ptr(), ws_bytes, _stream()))


def silu_and_mul(out: torch.Tensor, input: torch.Tensor) -> None:  # noqa: A002
    """csrc/ops.cpp:29-31. input [N, 2d] -> out [N, d], bf16."""
    _need_cuda(out, input)
    if input.dtype != torch.bfloat16 or out.dtype != torch.bfloat16:
        raise RuntimeError("silu_and_mul: bfloat16 only")
    assert input.is_contiguous() and out.is_contiguous()
    d = input.size(-1) // 2
    rows = input.numel() // (2 * d) if d else 0
    with torch.cuda.device(input.device):
        check(lib.moe_b200_silu_and_mul(out.data_ptr(), input.data_ptr(), rows, d, _stream()))


def swigluoai_and_mul(out: torch.Tensor, input: torch.Tensor, alpha: float = 1.702, limit: float = 7.0) -> None:  # noqa: A002
    """csrc/ops.cpp:33-36."""
    _need_cuda(out, input)
    if input.dtype != torch.bfloat16 or out.dtype != torch.bfloat16:
        raise RuntimeError("swigluoai_and_mul: bfloat16 only")
    assert input.is_contiguous() and out.is_contiguous()
    d = input.size(-1) // 2
    rows = input.numel() // (2 * d) if d else 0
    with torch.cuda.device(input.device):
        check(lib.moe_b200_swigluoai_and_mul(out.data_ptr(), input.data_ptr(), rows, d, alpha, limit, _stream()))


def moe_sum(input: torch.Tensor, output: torch.Tensor) -> None:  # noqa: A002
    """nanovllm/layers/for_moe/moe_easy_kernel.py:26-31. input [T, k, H] -> output [T, H], bf16."""
    _need_cuda(input, output)
    assert input.dtype == torch.bfloat16 and output.dtype == torch.bfloat16
    assert input.is_contiguous() and output.is_contiguous()
    T, k, H = input.shape
    with torch.cuda.device(input.device):
        check(lib.moe_b200_moe_sum(input.data_ptr(), output.data_ptr(), T, k, H, _stream()))


# ---------------------------------------------------------------- custom all-reduce (csrc/ops.cpp:77-95)
def meta_size() -> int:
    return int(lib.moe_b200_ar_meta_size())


def allocate_shared_buffer_and_handle(size: int) -> Tuple[int, bytes]:
    ptr = ctypes.c_int64(0)
    handle = (ctypes.c_uint8 * 64)()
    check(lib.moe_b200_ar_allocate_shared_buffer(size, ctypes.byref(ptr), handle))
    return int(ptr.value), bytes(handle)


def open_mem_handle(handle: bytes) -> int:
    buf = (ctypes.c_uint8 * 64).from_buffer_copy(bytes(handle))
    ptr = ctypes.c_int64(0)
    check(lib.moe_b200_ar_open_mem_handle(buf, ctypes.byref(ptr)))
    return int(ptr.value)


def close_mem_handle(ptr: int) -> None:
    """Unmaps a peer's buffer opened with open_mem_handle (the reference leaves this to process exit)."""
    check(lib.moe_b200_ar_close_mem_handle(int(ptr)))


def free_shared_buffer(ptr: int) -> None:
    check(lib.moe_b200_ar_free_shared_buffer(ptr))


def init_custom_ar(ipc_ptrs: List[int], rank_data: torch.Tensor, rank: int, fully_connected: bool) -> int:
    n = len(ipc_ptrs)
    arr = (ctypes.c_int64 * n)(*ipc_ptrs)
    h = ctypes.c_int64(0)
    with torch.cuda.device(rank_data.device):
        check(lib.moe_b200_ar_init(arr, n, rank_data.data_ptr(), rank_data.numel() * rank_data.element_size(), rank,
                                   int(fully_connected), ctypes.byref(h)))
    return int(h.value)


def dispose(fa: int) -> None:
    check(lib.moe_b200_ar_dispose(fa))


def register_buffer(fa: int, ipc_ptrs: List[int]) -> None:
    arr = (ctypes.c_int64 * len(ipc_ptrs))(*ipc_ptrs)
    check(lib.moe_b200_ar_register_buffer(fa, arr))


def register_fused_buffer(fa: int, ipc_ptrs: List[int], nbytes: int) -> None:
    """A second registered buffer, used only by the fused k-slot-sum + one-shot all-reduce (two halves in alternation,
    which saves that kernel its closing barrier). No reference counterpart."""
    arr = (ctypes.c_int64 * len(ipc_ptrs))(*ipc_ptrs)
    check(lib.moe_b200_ar_register_fused_buffer(fa, arr, nbytes))


def register_ll_buffer(fa: int, ipc_ptrs: List[int], nbytes: int) -> None:
    """The receive areas of the flag-in-data one-shot reduction (data and flag travel in the same 8 bytes, no
    barrier). No reference counterpart."""
    arr = (ctypes.c_int64 * len(ipc_ptrs))(*ipc_ptrs)
    check(lib.moe_b200_ar_register_ll_buffer(fa, arr, nbytes))


_AR_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def all_reduce(fa: int, inp: torch.Tensor, out: torch.Tensor, reg_buffer: int, reg_buffer_sz_bytes: int,
               algo: int = 0) -> None:
    _need_cuda(inp, out)
    if inp.dtype not in _AR_DTYPES or out.dtype != inp.dtype:
        raise RuntimeError("all_reduce: bf16/fp16/fp32 tensors of equal dtype only")
    if inp.numel() != out.numel():
        raise RuntimeError("all_reduce: input and output sizes differ")
    with torch.cuda.device(inp.device):
        check(lib.moe_b200_ar_all_reduce(fa, inp.data_ptr(), out.data_ptr(), inp.numel(), _AR_DTYPES[inp.dtype],
                                         reg_buffer, reg_buffer_sz_bytes, algo, status_word(inp.device).data_ptr(),
                                         _stream()))


def get_graph_buffer_ipc_meta(fa: int) -> Tuple[bytes, List[int]]:
    n = ctypes.c_int(0)
    check(lib.moe_b200_ar_graph_buffer_count(fa, ctypes.byref(n)))
    cnt = int(n.value)
    handles = (ctypes.c_uint8 * (64 * max(cnt, 1)))()
    offsets = (ctypes.c_int64 * max(cnt, 1))()
    check(lib.moe_b200_ar_get_graph_buffer_ipc_meta(fa, handles, offsets, cnt))
    return bytes(handles)[: 64 * cnt], [int(offsets[i]) for i in range(cnt)]


def register_graph_buffers(fa: int, handles: List[bytes], offsets: List[List[int]]) -> None:
    world = len(handles)
    cnt = len(offsets[0]) if offsets else 0
    flat_h = b"".join(bytes(h) for h in handles)
    hb = (ctypes.c_uint8 * max(len(flat_h), 1)).from_buffer_copy(flat_h if flat_h else b"\0")
    flat_o = [o for per_rank in offsets for o in per_rank]
    ob = (ctypes.c_int64 * max(len(flat_o), 1))(*flat_o) if flat_o else (ctypes.c_int64 * 1)()
    assert len(flat_h) == world * cnt * 64
    check(lib.moe_b200_ar_register_graph_buffers(fa, hb, ob, cnt))


__all__ = [
    "topk_softmax", "topk_softmax_renorm", "moe_align_block_size", "silu_and_mul", "swigluoai_and_mul", "moe_sum",
    "meta_size", "allocate_shared_buffer_and_handle", "open_mem_handle", "free_shared_buffer", "init_custom_ar",
    "dispose", "register_buffer", "all_reduce", "get_graph_buffer_ipc_meta", "register_graph_buffers",
    "status_word", "read_status", "rms_norm_quant_fp8", "add_rms_norm_quant_fp8", "w4_linear", "router_loss", "router_backward",
]
_ = _lib
