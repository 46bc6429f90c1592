"""Measured cases of the low-precision operators around the expert block and of the router's losses.

Four operators: the RMS norm whose output is e4m3 with scales ("norm"), products with 4-bit weights and group scales, dense
("w4_linear") and over the routed experts ("w4_experts"), and the router's balance and z losses with their gradients ("router").
`run` computes them in plain torch operations where `own` is false and by the framework's entry points where it is true.
"""
import math

import torch

own = False

FP8_MAX = 448.0
SCALE_FLOOR = 1e-10
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the norm in front of the experts of one decode batch, Qwen3-30B-A3B hidden size: launch and latency
        dict(name="norm_decode", op="norm", T=64, H=2048, group=128, residual=True, normed=True),
        # one layered-prefill batch at the hidden size of Qwen3-235B-A22B: bandwidth
        dict(name="norm_prefill", op="norm", T=8192, H=4096, group=128, residual=True, normed=True),
        # a final norm without a residual, one scale a token, a hidden size that is no multiple of 128
        dict(name="norm_token_odd", op="norm", T=1021, H=5000, group=-1, residual=False, normed=False),
        # attention output projection of one token (o_proj of Qwen3-30B-A3B: 32 heads x 128 -> 2048)
        dict(name="linear_one", op="w4_linear", M=1, N=2048, K=4096, group=128, zeros=False, bias=False),
        # the same layer of Qwen3-235B-A22B (64 heads x 128 -> 4096) for a decode batch, zero points, finer groups
        dict(name="linear_batch", op="w4_linear", M=16, N=4096, K=8192, group=64, zeros=True, bias=False),
        # a vocabulary projection: many output rows, an odd number of them, few tokens, the finest groups
        dict(name="linear_wide", op="w4_linear", M=5, N=131075, K=2048, group=32, zeros=False, bias=True),
        # the experts for a single token (Qwen3-30B-A3B): eight experts' weights, latency
        dict(name="experts_one", op="w4_experts", T=1, H=2048, E=128, k=8, I=768, group=128, zeros=False),
        # the benchmark's decode batch: nearly every expert is active, a few tokens each
        dict(name="experts_decode", op="w4_experts", T=64, H=2048, E=128, k=8, I=768, group=128, zeros=False),
        # the larger model's decode batch, odd batch size, zero points and finer groups
        dict(name="experts_large", op="w4_experts", T=93, H=4096, E=128, k=8, I=1536, group=64, zeros=True),
        # router losses of a small batch, bf16 logits: launches
        dict(name="router_small", op="router", T=64, E=128, k=8, dtype="bfloat16", masked=0.0),
        # one layered-prefill batch with padding at its end
        dict(name="router_prefill", op="router", T=8192, E=128, k=8, dtype="bfloat16", masked=0.1),
        # a training batch, fp32 logits, an expert count that is no power of two
        dict(name="router_train", op="router", T=65519, E=160, k=6, dtype="float32", masked=0.02),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "w4_linear", "w4_experts", "router"])
    if op == "norm":
        group = rng.choice([128, -1])
        h = 128 * rng.randint(2, 48) if group == 128 else 8 * _log(rng, 16, 768)
        t = _log(rng, 1, 8192 * 4096 // max(h, 4096))
        return dict(op=op, T=t, H=h, group=group, residual=rng.random() < 0.6, normed=rng.random() < 0.5)
    if op == "w4_linear":
        group = rng.choice([32, 64, 128])
        k = group * rng.randint(max(1, 256 // group), 8192 // group)
        n = _log(rng, 65, min(131075, 131075 * 2048 // k))
        return dict(op=op, M=_log(rng, 1, 24), N=n, K=k, group=group, zeros=rng.random() < 0.5, bias=rng.random() < 0.3)
    if op == "w4_experts":
        group = rng.choice([32, 64, 128])
        e = rng.choice([8, 16, 60, 64, 128])
        h = 128 * rng.randint(4, 32)
        i = 128 * rng.randint(2, 12)
        return dict(op=op, T=_log(rng, 1, 90), H=h, E=e, k=rng.choice([1, 2, 4, 6, 8]), I=i, group=group,
                    zeros=rng.random() < 0.5)
    e = rng.choice([8, 16, 60, 64, 100, 128, 160, 256, 384])
    return dict(op=op, T=_log(rng, 1, 65519 * 160 // max(e, 160)), E=e, k=rng.randint(1, 8),
                dtype=rng.choice(["bfloat16", "float32"]), masked=rng.choice([0.0, 0.1, 0.5]))


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _w4(g, group, zeros, *shape):
    """Packed 4-bit weights [..., N, K/2] (low nibble first), bf16 scales [..., N, K/group], zero points or None: bell-shaped
    codes and scales that differ by group, as a quantised layer has them."""
    *lead, n, k = shape
    codes = _randn(g, *lead, n, k // 2, 2, dtype=torch.bfloat16).mul_(2.7).round_().add_(8).clamp_(0, 15).to(torch.uint8)
    packed = codes[..., 0] | (codes[..., 1] << 4)
    del codes
    scale = (0.02 / 2.7 * torch.exp(0.3 * _randn(g, *lead, n, k // group))).to(torch.bfloat16)
    zp = None
    if zeros:
        zp = (_randn(g, *lead, n, k // group) + 8).round().clamp(0, 15).to(torch.uint8)
    return packed, scale, zp


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op = case["op"]
    if op == "norm":
        T, H, group = case["T"], case["H"], case["group"]
        s["x"] = _randn(g, T, H).to(torch.bfloat16)
        s["weight"] = (1 + 0.2 * _randn(g, H)).to(torch.bfloat16)
        # a residual stream a few layers deep: larger than the sublayer's output, a few outlier channels
        if case["residual"]:
            r = 3 * _randn(g, T, H)
            r[:, torch.randint(0, H, (4,), generator=g, device="cuda")] *= 12
            s["res"] = r.to(torch.bfloat16)
            s["res_out"] = torch.empty_like(s["res"])
        s["q"] = torch.empty(T, H, dtype=torch.float8_e4m3fn, device="cuda")
        s["scales"] = torch.empty(T, 1 if group < 0 else H // group, dtype=torch.float32, device="cuda")
        s["normed_out"] = torch.empty(T, H, dtype=torch.bfloat16, device="cuda") if case["normed"] else None
    elif op == "w4_linear":
        s["x"] = _randn(g, case["M"], case["K"]).to(torch.bfloat16)
        s["w"], s["s"], s["z"] = _w4(g, case["group"], case["zeros"], case["N"], case["K"])
        s["b"] = _randn(g, case["N"]).to(torch.bfloat16) if case["bias"] else None
        s["out"] = torch.empty(case["M"], case["N"], dtype=torch.bfloat16, device="cuda")
    elif op == "w4_experts":
        T, H, E, I = case["T"], case["H"], case["E"], case["I"]
        s["x"] = _randn(g, T, H).to(torch.bfloat16)
        s["w13"], s["s13"], s["z13"] = _w4(g, case["group"], case["zeros"], E, 2 * I, H)
        s["w2"], s["s2"], s["z2"] = _w4(g, case["group"], case["zeros"], E, H, I)
        p = torch.softmax(_randn(g, T, E), -1)
        top, ids = torch.topk(p, case["k"], -1)
        s["tw"], s["ids"] = top / top.sum(-1, keepdim=True), ids.to(torch.int32)
    else:
        T, E, k = case["T"], case["E"], case["k"]
        dt = getattr(torch, case["dtype"])
        s["logits"] = (1.5 * _randn(g, T, E) + _randn(g, E)).to(dt)
        s["ids"] = torch.topk(s["logits"].float(), k, -1)[1].to(torch.int32)
        s["mask"] = None
        if case["masked"] > 0:  # the padding at the batch's end
            s["mask"] = torch.arange(T, device="cuda") < T - int(case["masked"] * T)
        s["g_w"] = 0.1 * _randn(g, T, k)
        s["g_losses"] = torch.tensor([1e-2, 1e-3], device="cuda")
        s["losses"] = torch.empty(2, dtype=torch.float32, device="cuda")
        s["counts"] = torch.empty(E, dtype=torch.int32, device="cuda")
        s["num_tokens"] = torch.empty(1, dtype=torch.int32, device="cuda")
        s["mean_probs"] = torch.empty(E, dtype=torch.float32, device="cuda")
        s["g_logits"] = torch.empty_like(s["logits"])
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from layered_prefill_b200 import fused_moe, ops
    op = s["op"]
    if op == "norm":
        if s["residual"]:
            ops.add_rms_norm_quant_fp8(s["q"], s["scales"], s["res"], s["x"], s["weight"], EPS, group_size=s["group"],
                                       normed_out=s["normed_out"], residual_out=s["res_out"])
        else:
            ops.rms_norm_quant_fp8(s["q"], s["scales"], s["x"], s["weight"], EPS, group_size=s["group"],
                                   normed_out=s["normed_out"])
        return [s["q"], s["scales"]] + ([s["res_out"]] if s["residual"] else []) + ([s["normed_out"]] if s["normed"] else [])
    if op == "w4_linear":
        ops.w4_linear(s["out"], s["x"], s["w"], s["s"], s["z"], s["b"])
        return s["out"]
    if op == "w4_experts":
        return fused_moe.fused_experts(s["x"], s["w13"], s["w2"], None, None, s["tw"], s["ids"], w1_scale=s["s13"],
                                       w2_scale=s["s2"], w1_zp=s["z13"], w2_zp=s["z2"], block_shape=[0, s["group"]])
    ops.router_loss(s["losses"], s["counts"], s["num_tokens"], s["mean_probs"], s["logits"], s["ids"], s["mask"])
    ops.router_backward(s["g_logits"], s["logits"], s["ids"], s["counts"], s["num_tokens"], s["g_losses"], s["g_w"], True,
                        s["mask"])
    return [s["losses"], s["counts"], s["num_tokens"], s["mean_probs"], s["g_logits"]]


def _dequant(packed, scale, zp, group):
    """fp32 [..., N, K] of packed 4-bit weights."""
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).float()
    codes = codes.unflatten(-1, (-1, group))
    zero = 8.0 if zp is None else zp.float()[..., None]
    return ((codes - zero) * scale.float()[..., None]).flatten(-2)


def _plain(s):
    op = s["op"]
    if op == "norm":
        x = s["x"].float()
        outs = []
        if s["residual"]:
            r = (x + s["res"].float()).to(torch.bfloat16)  # the residual stream as it is stored is what is normalised
            x = r.float()
            outs.append(r)
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"].float()
        if s["normed"]:
            outs.append(y.to(torch.bfloat16))
        groups = y.unflatten(-1, (-1, s["group"] if s["group"] > 0 else s["H"]))
        scale = groups.abs().amax(-1).clamp(min=SCALE_FLOOR) / FP8_MAX
        q = (groups / scale[..., None]).flatten(-2).to(torch.float8_e4m3fn)
        return [q, scale] + outs
    if op == "w4_linear":
        y = s["x"].float() @ _dequant(s["w"], s["s"], s["z"], s["group"]).t()
        if s["b"] is not None:
            y = y + s["b"].float()
        return y.to(torch.bfloat16)
    if op == "w4_experts":
        T, E, k = s["T"], s["E"], s["k"]
        x, w13, w2 = s["x"].float(), (s["w13"], s["s13"], s["z13"]), (s["w2"], s["s2"], s["z2"])
        if T * k < E:  # few slots: the weights of each slot's expert
            e = s["ids"].flatten().long()
            x = x.repeat_interleave(k, 0)[:, None, :]
            w13, w2 = ([None if v is None else v[e] for v in w] for w in (w13, w2))
        # otherwise every expert on every token, of which the routed ones are weighted
        gate, up = torch.matmul(x, _dequant(*w13, s["group"]).transpose(1, 2)).chunk(2, -1)
        h = gate * torch.sigmoid(gate) * up
        y = torch.bmm(h, _dequant(*w2, s["group"]).transpose(1, 2))  # [slots, 1, H] or [E, T, H]
        if T * k < E:
            return (y.view(T, k, -1) * s["tw"][..., None]).sum(1).to(torch.bfloat16)
        w = torch.zeros(T, E, device=x.device).scatter_add_(1, s["ids"].long(), s["tw"])
        return (y * w.t()[..., None]).sum(0).to(torch.bfloat16)
    logits = s["logits"].float()
    E, k = s["E"], s["k"]
    keep = torch.ones(s["T"], device=logits.device) if s["mask"] is None else s["mask"].float()
    ids = s["ids"].long()
    num = keep.sum()
    n = num.clamp(min=1)
    lse = torch.logsumexp(logits, -1)
    p = torch.exp(logits - lse[:, None])
    counts = torch.zeros(E, device=logits.device).scatter_add_(0, ids.flatten(), keep.repeat_interleave(k))
    mean_probs = (p * keep[:, None]).double().sum(0) / n
    balance = E * (counts / n * mean_probs).sum()
    z = (lse * lse * keep).double().sum() / n
    # backward: of the losses through p and lse, and of the renormalised routed weights through p
    picked = p.gather(1, ids)
    total = picked.sum(-1, keepdim=True)
    w = picked / total
    du = (s["g_w"] - (s["g_w"] * w).sum(-1, keepdim=True)) / total
    u = (s["g_losses"][0] * E / (n * n) * counts).expand_as(p).scatter_add(1, ids, du)
    grad = p * (u - (p * u).sum(-1, keepdim=True) + s["g_losses"][1] * 2 * lse[:, None] / n)
    grad = torch.where(keep[:, None] > 0, grad, torch.zeros_like(grad))
    return [torch.stack((balance, z)).float(), counts.to(torch.int32), num.to(torch.int32).reshape(1), mean_probs.float(),
            grad.to(s["logits"].dtype)]


# ---------------------------------------------------------------------------------------------------- least work
def work(case):
    op = case["op"]
    if op == "norm":
        T, H = case["T"], case["H"]
        n_scales = T * (1 if case["group"] < 0 else H // case["group"])
        per = 2 + 1 + (4 if case["residual"] else 0) + (2 if case["normed"] else 0)
        return {"bytes": T * H * per + 2 * H + 4 * n_scales, "flops": 8 * T * H}
    if op == "w4_linear":
        M, N, K = case["M"], case["N"], case["K"]
        per_group = 2 + (1 if case["zeros"] else 0)
        return {"bytes": N * K // 2 + N * (K // case["group"]) * per_group + 2 * M * (K + N) + (2 * N if case["bias"] else 0),
                "flops": 2 * M * N * K}
    if op == "w4_experts":
        T, H, E, k, I = (case[c] for c in ("T", "H", "E", "k", "I"))
        active = E * (1 - (1 - k / E) ** T)  # expected number of experts with a token
        per_group = 2 + (1 if case["zeros"] else 0)
        expert = 3 * H * I / 2 + 3 * H * I / case["group"] * per_group
        return {"bytes": active * expert + 4 * T * H + 8 * T * k, "flops": 2 * T * k * 3 * H * I}
    T, E, k = case["T"], case["E"], case["k"]
    b = 2 if case["dtype"] == "bfloat16" else 4
    # logits, ids and the weights' gradients come in, the gradient goes out
    return {"bytes": 2 * T * E * b + 8 * T * k + (T if case["masked"] else 0) + 8 * E, "flops": 12 * T * E}


# ---------------------------------------------------------------------------------------------------- 64 bits
def _codes64(packed):
    out = torch.empty(*packed.shape[:-1], 2 * packed.shape[-1], dtype=torch.float64, device=packed.device)
    out[..., 0::2] = (packed % 16).double()
    out[..., 1::2] = (packed // 16).double()
    return out


def _weight64(packed, scale, zp, group):
    w = _codes64(packed)
    s = scale.double().repeat_interleave(group, -1)
    return w.sub_(8 if zp is None else zp.double().repeat_interleave(group, -1)).mul_(s)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        v = s["x"].double()
        tail = []
        if case["residual"]:
            v = v + s["res"].double()
            tail.append(v)
            v = v.to(torch.bfloat16).double()
        y = v / torch.sqrt(v.pow(2).sum(-1, keepdim=True) / case["H"] + EPS) * s["weight"].double()
        if case["normed"]:
            tail.append(y)
        width = case["H"] if case["group"] < 0 else case["group"]
        amax = y.view(case["T"], -1, width).abs().max(-1).values
        scale = torch.maximum(amax, torch.full_like(amax, SCALE_FLOOR)) / FP8_MAX
        return [y / scale.repeat_interleave(width, -1), scale] + tail
    if op == "w4_linear":
        rows = []
        step = max(1, (1 << 28) // case["K"])
        for a in range(0, case["N"], step):
            b = min(case["N"], a + step)
            w = _weight64(s["w"][a:b], s["s"][a:b], None if s["z"] is None else s["z"][a:b], case["group"])
            rows.append(torch.einsum("mk,nk->mn", s["x"].double(), w))
        y = torch.cat(rows, 1)
        return y if s["b"] is None else y + s["b"].double()
    if op == "w4_experts":
        out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
        I = case["I"]
        for e in range(case["E"]):
            t, j = torch.nonzero(s["ids"] == e, as_tuple=True)
            if t.numel() == 0:
                continue
            zp = (None, None) if s["z13"] is None else (s["z13"][e], s["z2"][e])
            gu = s["x"][t].double() @ _weight64(s["w13"][e], s["s13"][e], zp[0], case["group"]).T
            a, b = gu[:, :I], gu[:, I:]
            h = a / (1 + torch.exp(-a)) * b
            y = h @ _weight64(s["w2"][e], s["s2"][e], zp[1], case["group"]).T
            out.index_add_(0, t, y * s["tw"][t, j].double()[:, None])
        return out
    E, T = case["E"], case["T"]
    live = torch.arange(T, device="cuda") if s["mask"] is None else torch.nonzero(s["mask"])[:, 0]
    n = max(1, live.numel())
    leaf = s["logits"][live].double().requires_grad_(True)
    ids = s["ids"][live].long()
    p = torch.softmax(leaf, -1)
    lse = torch.logsumexp(leaf, -1)
    counts = torch.bincount(ids.flatten(), minlength=E).double()
    mean_probs = p.sum(0) / n
    balance = E * torch.dot(counts / n, mean_probs)
    z = lse.square().sum() / n
    picked = p.gather(1, ids)
    w = picked / picked.sum(-1, keepdim=True)
    g = s["g_losses"].double()
    (balance * g[0] + z * g[1] + (w * s["g_w"][live].double()).sum()).backward()
    grad = torch.zeros(T, E, dtype=torch.float64, device="cuda")
    grad[live] = leaf.grad
    return [torch.stack((balance, z)).detach(), None, None, mean_probs.detach(), grad]
