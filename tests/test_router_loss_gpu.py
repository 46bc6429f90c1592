"""Router losses, counts and gradients against autograd in 64 bits, and the gradient against differences.

Tolerances. The logits here stay within 30 of their row's maximum: the exponent's argument is off by 30 * 1.45 * 2^-24, so p by 2^-18 of
itself with the sum and the reciprocal included; sums over tokens are short fp32 chains joined in 64 bits. So the losses and the mean
probabilities are within 2^-17 and a gradient within 2^-16 of sum of the magnitudes of its terms, and its rounding (2^-8 for bf16,
2^-24 for fp32 of the value) comes on top."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(T, E, k, dtype, seed, masked=0.0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    logits = (scale * torch.randn(T, E, generator=g).clamp(-4, 4) + torch.randn(E, generator=g)).to(dtype)
    ids = torch.topk(logits.float(), k, -1)[1].to(torch.int32)
    mask = torch.rand(T, generator=g) >= masked if masked else None
    g_w = torch.randn(T, k, generator=g)
    g_l = torch.tensor([0.7, -0.3])
    return [None if t is None else t.cuda() for t in (logits, ids, mask, g_w, g_l)]


def _run(logits, ids, mask, g_w, g_l, renorm=True):
    from layered_prefill_b200 import ops
    T, E = logits.shape
    dev = logits.device
    losses, mean = torch.empty(2, device=dev), torch.empty(E, device=dev)
    counts, n = torch.empty(E, dtype=torch.int32, device=dev), torch.empty(1, dtype=torch.int32, device=dev)
    ops.router_loss(losses, counts, n, mean, logits, ids, mask)
    grad = torch.full_like(logits, float("nan"))
    ops.router_backward(grad, logits, ids, counts, n, g_l, g_w, renorm, mask)
    return losses, counts, n, mean, grad


def _oracle(logits, ids, mask, g_w, g_l, renorm=True):
    T, E = logits.shape
    live = torch.arange(T, device=logits.device) if mask is None else torch.nonzero(mask)[:, 0]
    n = max(1, live.numel())
    leaf = logits[live].double().requires_grad_(True)
    p, lse = torch.softmax(leaf, -1), torch.logsumexp(leaf, -1)
    ok = (ids[live] >= 0) & (ids[live] < E)
    idx = ids[live].long().clamp(0, E - 1)
    counts = torch.zeros(E, dtype=torch.float64, device=logits.device).scatter_add_(0, idx.flatten(), ok.flatten().double())
    mean = p.sum(0) / n
    losses = torch.stack((E * (counts / n * mean).sum(), lse.square().sum() / n))
    picked = p.gather(1, idx) * ok
    w = picked / picked.sum(-1, keepdim=True) if renorm else picked
    total = leaf.sum() * 0
    size = torch.zeros(T, E, dtype=torch.float64, device=logits.device)
    u = torch.zeros(live.numel(), E, dtype=torch.float64, device=logits.device)
    if g_l is not None:
        total = total + (losses * g_l.double()).sum()
        u = u + g_l[0].double().abs() * E * counts / n / n + (g_l[1].double().abs() * 2 * lse.detach().abs() / n)[:, None]
    if g_w is not None:
        gw = g_w[live].double()
        total = total + torch.where(ok, w * gw, torch.zeros_like(w)).sum()
        s = picked.detach().sum(-1, keepdim=True) if renorm else 1.0
        u = u.scatter_add(1, idx, (gw.abs() + ((gw * w.detach()).abs().sum(-1, keepdim=True) if renorm else 0)) / s * ok)
    total.backward()
    grad = torch.zeros(T, E, dtype=torch.float64, device=logits.device)
    grad[live] = leaf.grad
    pd = p.detach()
    size[live] = pd * (u + (pd * u).sum(-1, keepdim=True))
    return losses.detach(), counts, live.numel(), mean.detach(), grad, size


def _check(got, want, dtype):
    losses, counts, n, mean, grad = got
    losses64, counts64, n64, mean64, grad64, size = want
    assert int(n) == n64 and torch.equal(counts.double(), counts64)
    assert ((losses.double() - losses64).abs() <= 2.0 ** -17 * losses64.abs()).all(), (losses, losses64)
    assert ((mean.double() - mean64).abs() <= 2.0 ** -17 * mean64).all()
    eps = torch.finfo(dtype).eps / 2
    bound = 1.01 * eps * grad64.abs() + 2.0 ** -16 * size + 1e-38
    assert ((grad.double() - grad64).abs() <= bound).all(), ((grad.double() - grad64).abs() / bound).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 128, 8), (2, 8, 8), (3, 33, 5), (64, 128, 8), (17, 60, 4), (100, 100, 7),
                                   (513, 160, 6), (1000, 256, 8), (129, 384, 3), (70, 1024, 33), (40, 512, 40), (4099, 64, 2)])
def test_losses_counts_and_gradients(T, E, k, dtype):
    args = _inputs(T, E, k, dtype, T + E)
    for renorm in (True, False):
        _check(_run(*args, renorm), _oracle(*args, renorm), dtype)


@pytest.mark.parametrize("T,E,k", [(5, 1024, 8), (16, 1024, 1024), (16, 1001, 3), (128, 128, 128), (129, 127, 9), (17, 1023, 200)])
def test_sizes_at_the_edges_of_the_shapes(T, E, k):
    for dtype in (torch.bfloat16, torch.float32):
        args = _inputs(T, E, k, dtype, T * E, masked=0.2)
        for renorm in (True, False):
            _check(_run(*args, renorm), _oracle(*args, renorm), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_tokens_count_for_nothing_whatever_they_hold(dtype):
    logits, ids, mask, g_w, g_l = _inputs(300, 96, 4, dtype, 1, masked=0.4)
    want = _oracle(logits, ids, mask, g_w, g_l)
    dead = torch.nonzero(~mask)[:, 0]
    logits[dead[0]], logits[dead[1]], logits[dead[2]] = float("nan"), float("inf"), float("-inf")
    ids[dead[3]] = 10 ** 9
    g_w[dead[4]] = float("nan")
    got = _run(logits, ids, mask, g_w, g_l)
    _check(got, want, dtype)
    assert (got[4][dead] == 0).all()
    same = _run(logits, ids, mask.to(torch.uint8) * 7, g_w, g_l)
    assert all(torch.equal(a, b) for a, b in zip(got, same))


def test_offsets_past_32_bits():
    T, E, k, n = 2**22 + 101, 1024, 2, 60
    part = _inputs(2 * n, E, k, torch.bfloat16, 11)
    ends = torch.cat((torch.arange(n), torch.arange(T - n, T))).cuda()
    logits = torch.full((T, E), float("nan"), dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(T, k, dtype=torch.int32, device="cuda")
    mask = torch.zeros(T, dtype=torch.bool, device="cuda")
    g_w = torch.zeros(T, k, device="cuda")
    logits[ends], ids[ends], mask[ends], g_w[ends] = part[0], part[1], True, part[3]
    losses, counts, live, mean, grad = _run(logits, ids, mask, g_w, part[4])
    assert not grad[n:-n].any()
    _check((losses, counts, live, mean, grad[ends]), _oracle(*part), torch.bfloat16)


def test_no_token_counts():
    logits, ids, _, g_w, g_l = _inputs(20, 16, 2, torch.float32, 2)
    losses, counts, n, mean, grad = _run(logits, ids, torch.zeros(20, dtype=torch.bool, device="cuda"), g_w, g_l)
    assert (losses == 0).all() and (counts == 0).all() and int(n) == 0 and (mean == 0).all() and (grad == 0).all()
    losses, counts, n, mean, grad = _run(logits[:0], ids[:0], None, g_w[:0], g_l)
    assert (losses == 0).all() and (counts == 0).all() and int(n) == 0 and (mean == 0).all() and grad.shape == (0, 16)


def test_masked_experts_and_ids_outside():
    logits, ids, _, g_w, g_l = _inputs(50, 40, 3, torch.float32, 3)
    logits[:, 5:9] = float("-inf")              # experts that are switched off
    ids = torch.topk(logits, 3, -1)[1].to(torch.int32)
    ids[7, 1], ids[8, 0] = -1, 40
    ids[9] = ids[9, 0]                          # the same expert three times
    got, want = _run(logits, ids, None, g_w, g_l), _oracle(logits, ids, None, g_w, g_l)
    _check(got, want, torch.float32)
    assert (got[4][:, 5:9] == 0).all()


def test_one_gradient_at_a_time():
    logits, ids, mask, g_w, g_l = _inputs(80, 64, 4, torch.float32, 4, masked=0.2)
    for a in ((mask, g_w, None), (mask, None, g_l), (None, None, None)):
        got = _run(logits, ids, *a)
        _check(got, _oracle(logits, ids, *a), torch.float32)


def test_balanced_routing_has_a_loss_of_k():
    E, k = 32, 4
    logits = torch.zeros(64, E, device="cuda")
    ids = ((torch.arange(64)[:, None] * k + torch.arange(k)) % E).to(torch.int32).cuda()
    losses, counts, _, mean, _ = _run(logits, ids, None, None, None)
    assert abs(float(losses[0]) - k) < 1e-5 and (counts == 64 * k // E).all()


def test_two_runs_give_the_same_bits():
    args = _inputs(5000, 200, 6, torch.float32, 6, masked=0.1)
    a = _run(*args)
    for _ in range(3):
        assert all(torch.equal(u, v) for u, v in zip(a, _run(*args)))


@pytest.mark.parametrize("renorm", [True, False])
def test_autograd_of_the_router_and_differences(renorm):
    """fused_topk_with_loss in a graph with a gate weight; and the gradient against central differences of the 64-bit loss."""
    from layered_prefill_b200 import fused_moe
    T, H, E, k = 30, 32, 16, 3
    g = torch.Generator().manual_seed(7)
    x = torch.randn(T, H, generator=g).cuda()
    gate = (torch.randn(E, H, generator=g) * 0.4).cuda().requires_grad_(True)
    mask = (torch.arange(T) < 25).cuda()
    g_w = torch.randn(T, k, generator=g).cuda()
    logits = x @ gate.t()
    logits.retain_grad()
    tw, ti, balance, z, counts = fused_moe.fused_topk_with_loss(logits, k, renorm, mask)
    want_tw, want_ti, _ = fused_moe.fused_topk(x, logits.detach(), k, renorm)
    assert torch.equal(tw, want_tw) and torch.equal(ti, want_ti)
    assert not counts.requires_grad and not ti.requires_grad
    loss = 0.5 * balance + 0.25 * z + (tw * g_w).sum()
    loss.backward()
    want = _oracle(logits.detach(), ti, mask, g_w, torch.tensor([0.5, 0.25], device="cuda"), renorm)
    assert ((logits.grad.double() - want[4]).abs() <= 2.0 ** -15 * want[5] + 1e-38).all()
    assert torch.allclose(gate.grad, logits.grad.t() @ x, rtol=1e-4, atol=1e-6)

    def f(l):
        p, lse = torch.softmax(l, -1), torch.logsumexp(l, -1)
        picked = p.gather(1, ti.long())
        w = picked / picked.sum(-1, keepdim=True) if renorm else picked
        keep = mask.double()
        bal = E * (counts.double() / 25 * (p * keep[:, None]).sum(0) / 25).sum()
        return 0.5 * bal + 0.25 * (lse.square() * keep).sum() / 25 + (w * g_w.double() * keep[:, None]).sum()

    base, h = logits.detach().double(), 1e-5
    for t, e in ((0, 0), (3, 7), (24, int(ti[24, 0])), (10, int(ti[10, 2])), (26, 4)):
        d = torch.zeros_like(base)
        d[t, e] = h
        diff = float(f(base + d) - f(base - d)) / (2 * h)
        assert abs(diff - float(logits.grad[t, e])) < 1e-5, (t, e)


def test_autograd_parts_that_take_no_part():
    from layered_prefill_b200 import fused_moe
    logits = torch.randn(8, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    tw, ti, balance, z, counts = fused_moe.fused_topk_with_loss(logits, 2, True)
    (g,) = torch.autograd.grad(tw.sum(), logits, retain_graph=True)  # renormalised weights sum to one
    assert g.float().abs().max() < 1e-6
    (g,) = torch.autograd.grad(z, logits)
    assert g.float().abs().max() > 0
    strided = torch.randn(16, 8, device="cuda").t().requires_grad_(True)
    fused_moe.fused_topk_with_loss(strided, 2, False)[2].backward()
    assert strided.grad.shape == strided.shape
    with pytest.raises(RuntimeError):
        fused_moe.fused_topk_with_loss(logits, 17, True)
    with pytest.raises(RuntimeError):
        fused_moe.fused_topk_with_loss(logits.detach().cpu(), 2, True)


def test_a_captured_training_step_replays():
    from layered_prefill_b200 import fused_moe
    static = torch.randn(64, 32, device="cuda")

    def step():
        leaf = static.detach().requires_grad_(True)
        tw, ti, balance, z, counts = fused_moe.fused_topk_with_loss(leaf, 4, True)
        return torch.autograd.grad(balance + 0.1 * z + tw[:, 0].sum(), leaf)[0], counts

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad, counts = step()
    static.copy_(torch.randn(64, 32, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    want, want_counts = step()
    assert torch.equal(grad, want) and torch.equal(counts, want_counts)


def test_refusals():
    from layered_prefill_b200 import ops
    from layered_prefill_b200._lib import MoeB200Error
    logits, ids, mask, g_w, g_l = _inputs(10, 16, 2, torch.float32, 1)
    o = dict(losses=torch.empty(2, device="cuda"), counts=torch.empty(16, dtype=torch.int32, device="cuda"),
             num_tokens=torch.empty(1, dtype=torch.int32, device="cuda"), mean_probs=torch.empty(16, device="cuda"),
             gating_output=logits, topk_ids=ids)
    for bad in (dict(topk_ids=ids.long()), dict(gating_output=logits.half()), dict(gating_output=logits.cpu()),
                dict(counts=o["counts"].float()), dict(losses=torch.empty(3, device="cuda")), dict(topk_ids=ids[:5]),
                dict(token_mask=torch.ones(9, dtype=torch.bool, device="cuda")), dict(token_mask=torch.ones(10, device="cuda")),
                dict(gating_output=logits.t().contiguous().t())):
        with pytest.raises(RuntimeError):
            ops.router_loss(**{**o, **bad})
    big = torch.zeros(2, 1025, device="cuda")
    with pytest.raises(MoeB200Error):
        ops.router_loss(o["losses"], torch.empty(1025, dtype=torch.int32, device="cuda"), o["num_tokens"],
                        torch.empty(1025, device="cuda"), big, ids[:2])
    with pytest.raises(RuntimeError):
        ops.router_backward(torch.empty_like(logits).bfloat16(), logits, ids, o["counts"], o["num_tokens"], g_l, g_w, True)


_FRESH = """
import sys
sys.path.insert(0, {root!r})
import torch
from tests.test_router_loss_gpu import _check, _inputs, _oracle, _run
failed = []
for T, E in {shapes!r}:
    for dtype in (torch.bfloat16, torch.float32):
        args = _inputs(T, E, 3, dtype, T + E)
        try:
            _check(_run(*args), _oracle(*args), dtype)
        except Exception as e:
            failed.append((T, E, str(dtype), str(e)[:200]))
assert not failed, failed
print("OK")
"""


@pytest.mark.parametrize("shapes", [((50, 288), (32, 320), (16, 372), (300, 576), (300, 640), (300, 720)),
                                    ((50, 277), (16, 371), (300, 577), (300, 721))])
def test_shared_memory_just_below_48_kb_in_a_process_of_its_own(shapes):
    """132 E bytes (one CTA) or 68 E (several) of dynamic shared memory below 48 KB that pass it with the kernel's own arrays. What
    a kernel may take stays set in a process, so no larger call may come before: sizes ascend, E in vectors and not."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _FRESH.format(root=root, shapes=shapes)], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "OK" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("T,E", [(2**27, 8), (2**23, 260)])
def test_long_batches_keep_their_precision(T, E):
    """Millions of equal tokens: every addition rounds the same way, so that one chain of fp32 additions over all of a lane's tokens
    (7085 and 1772 of them) is off by more than 2^-17. All tokens being equal, mean_probs is the softmax of one of them."""
    from layered_prefill_b200 import ops
    g = torch.Generator().manual_seed(E)
    row = torch.randn(E, generator=g).to(torch.bfloat16).cuda()
    logits = row.expand(T, E).contiguous()
    ids = torch.full((T, 1), 3, dtype=torch.int32, device="cuda")
    losses, mean = torch.empty(2, device="cuda"), torch.empty(E, device="cuda")
    counts, n = torch.empty(E, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
    ops.router_loss(losses, counts, n, mean, logits, ids)
    p, lse = torch.softmax(row.double(), -1), torch.logsumexp(row.double(), -1)
    assert int(n) == T and int(counts[3]) == T and int(counts.sum()) == T
    assert ((mean.double() - p).abs() <= 2.0 ** -17 * p).all(), ((mean.double() - p).abs() / p).max()
    want = torch.stack((E * p[3], lse.square()))
    assert ((losses.double() - want).abs() <= 2.0 ** -17 * want).all(), (losses, want)


def test_two_host_threads_with_different_numbers_of_experts():
    """Each on its own stream; the amounts of shared memory differ, the same bits come back every time."""
    import threading
    cases = [_inputs(16, 1000, 3, torch.float32, 1), _inputs(40, 300, 3, torch.float32, 2), _inputs(900, 600, 3, torch.float32, 3)]
    want = [_run(*c) for c in cases]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got = _run(*cases[i])
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        except BaseException as e:  # noqa: BLE001
            failed.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("E", [4, 28, 32, 36, 64, 68, 92, 96, 100, 132, 164, 188, 192, 196, 220, 224, 228, 252, 256])
def test_every_number_of_vectors_a_lane(E):
    for T, dtype in ((45, torch.bfloat16), (700, torch.float32)):
        args = _inputs(T, E, min(E, 6), dtype, T + E, masked=0.1)
        _check(_run(*args), _oracle(*args), dtype)
        _check(_run(args[0], args[1], args[2], None, args[4]), _oracle(args[0], args[1], args[2], None, args[4]), dtype)
