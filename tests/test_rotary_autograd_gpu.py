"""The rotary embedding's derivative: what it refuses, weights that are used twice or whose gradient moves (GPU)."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from meshy_b200.ops.rotary import Rope, qkv_rotary

pytestmark = pytest.mark.gpu
Hq, Hkv, HD = 4, 2, 64
ROPE = Rope(HD, 1e4)


def _inputs(T=37, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * HD, generator=g, device="cuda").bfloat16()
    w = [(1 + 0.2 * torch.randn(HD, generator=g, device="cuda")).bfloat16() for _ in range(2)]
    grads = [torch.randn(T, h, HD, generator=g, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv)]
    return qkv, torch.arange(T, dtype=torch.int32, device="cuda") * 3, w, grads


@pytest.mark.parametrize("which", ["qkv", "q_norm", "k_norm"])
@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("requires_grad", [True, False])
def test_forward_mode_is_refused(which, grad_mode, requires_grad):
    """A tangent must not vanish in silence, whether or not a backward pass is recorded."""
    qkv, pos, (wq, wk), _ = _inputs()
    args = {"qkv": qkv, "q_norm": wq, "k_norm": wk}
    if requires_grad:
        args["qkv"].requires_grad_()
    with fwAD.dual_level(), torch.set_grad_enabled(grad_mode):
        args[which] = fwAD.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode|jvp"):
            qkv_rotary(args["qkv"], pos, ROPE, Hq, Hkv, args["q_norm"], args["k_norm"])
        # tensors without a tangent are served inside a dual level as well
        qkv_rotary(_inputs()[0], pos, ROPE, Hq, Hkv, wq, wk)


def _plain(w, inputs, w2=None):
    """The gradients of the norms' weights without a ``main_grad``."""
    qkv, pos, _, grads = inputs
    leaves = [w.clone().requires_grad_(), (w if w2 is None else w2).clone().requires_grad_()]
    return torch.autograd.grad(qkv_rotary(qkv, pos, ROPE, Hq, Hkv, *leaves), leaves, grads)


@pytest.mark.parametrize("when", ["given", "moved", "taken away"])
def test_main_grad_is_looked_up_in_the_backward_pass(when):
    """As the other operators do: a trainer may hand the buffers out, swap or drop them after the forward pass."""
    inputs = _inputs()
    qkv, pos, weights, grads = inputs
    want = _plain(weights[0], inputs, weights[1])
    w = [x.clone().requires_grad_() for x in weights]
    early, late = ([torch.full((HD,), 3.0, device="cuda") for _ in w] for _ in range(2))
    if when != "given":
        for x, m in zip(w, early):
            x.main_grad = m
    out = qkv_rotary(qkv, pos, ROPE, Hq, Hkv, *w)
    for x, m in zip(w, late):
        x.main_grad = None if when == "taken away" else m
    torch.autograd.backward(out, grads)
    assert all(bool((m == 3.0).all()) for m in early)
    for x, m, g in zip(w, late, want):
        if when == "taken away":
            assert torch.equal(x.grad, g) and bool((m == 3.0).all())
        else:  # (the gradient in bf16 is the same sum rounded once more; adding 3 and taking it off again rounds in fp32)
            assert x.grad is None
            assert bool(((m - 3.0 - g.float()).abs() <= 2.0 ** -8 * g.float().abs() + 2.0 ** -23 * (m.abs() + 3)).all())


@pytest.mark.parametrize("T", [1, 37, 5003, 0])
@pytest.mark.parametrize("hd", [64, 176])
def test_one_weight_for_queries_and_keys(T, hd):
    """Tied norms: their ``main_grad`` gets both sums, whatever the timing."""
    rope = Rope(hd, 1e4)
    g = torch.Generator(device="cuda").manual_seed(T)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * hd, generator=g, device="cuda").bfloat16()
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    w = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).bfloat16()
    grads = [torch.randn(T, h, hd, generator=g, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv)]

    def run(*leaves):
        torch.autograd.backward(qkv_rotary(qkv, pos, rope, Hq, Hkv, *leaves), grads)

    apart = [w.clone().requires_grad_() for _ in range(2)]
    for x in apart:
        x.main_grad = torch.zeros(hd, device="cuda")
    run(*apart)
    tied = w.clone().requires_grad_()
    tied.main_grad = torch.zeros(hd, device="cuda")
    for _ in range(20):
        tied.main_grad.zero_()
        run(tied, tied)
        assert tied.grad is None and torch.equal(tied.main_grad, apart[0].main_grad + apart[1].main_grad)
    # two weights whose buffers are one
    for x in apart:
        x.main_grad = tied.main_grad
    tied.main_grad.zero_()
    run(*apart)
    torch.cuda.synchronize()
    total = tied.main_grad.clone()
    tied.main_grad.zero_()
    run(tied, tied)
    assert torch.equal(total, tied.main_grad)
    # without one, autograd adds the two up
    free = w.clone().requires_grad_()
    run(free, free)
    lone = [w.clone().requires_grad_() for _ in range(2)]
    run(*lone)
    assert torch.equal(free.grad, lone[0].grad + lone[1].grad)


@pytest.mark.parametrize("reentrant", [True, False])
def test_recomputed_and_repeated_backward_passes(reentrant):
    """Activation checkpointing gives the plain pass's gradients; a second pass over a kept graph adds them once more."""
    from torch.utils.checkpoint import checkpoint

    qkv, pos, weights, grads = _inputs(T=300)

    def run(wrap):
        x, w = qkv.clone().requires_grad_(), [y.clone().requires_grad_() for y in weights]
        for y in w:
            y.main_grad = torch.zeros(HD, device="cuda")
        f = lambda x: qkv_rotary(x, pos, ROPE, Hq, Hkv, *w)  # noqa: E731  (a module's own weights)
        out = checkpoint(f, x, use_reentrant=reentrant) if wrap else f(x)
        torch.autograd.backward(out, grads, retain_graph=not wrap)
        return x, w, out

    x, w, out = run(False)
    y, v, _ = run(True)
    assert torch.equal(x.grad, y.grad) and all(torch.equal(a.main_grad, b.main_grad) for a, b in zip(w, v))
    assert all(a.grad is None for a in w + v)
    once = [a.main_grad.clone() for a in w]
    torch.autograd.backward(out, grads)
    assert all(torch.equal(a.main_grad, 2 * b) for a, b in zip(w, once))


def test_backward_passes_of_several_threads():
    """The passes look the weights' buffers up under Python's lock, from autograd's thread."""
    import threading

    wrong = []

    def work(i):
        try:
            inputs = _inputs(seed=i)
            want = _plain(inputs[2][0], inputs, inputs[2][1])
            for _ in range(30):
                w = [y.clone().requires_grad_() for y in inputs[2]]
                for y in w:
                    y.main_grad = torch.zeros(HD, device="cuda")
                torch.autograd.backward(qkv_rotary(inputs[0], inputs[1], ROPE, Hq, Hkv, *w), inputs[3])
                torch.cuda.synchronize()
                if not all(torch.equal(y.main_grad.bfloat16(), g) for y, g in zip(w, want)):
                    wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads) and not wrong, wrong


def test_a_captured_backward_pass_adds_to_main_grad():
    qkv, pos, weights, grads = _inputs(T=64)
    w = [y.clone().requires_grad_() for y in weights]
    for y in w:
        y.main_grad = torch.zeros(HD, device="cuda")

    def step():
        torch.autograd.backward(qkv_rotary(qkv, pos, ROPE, Hq, Hkv, *w), grads)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    once = [y.main_grad.clone() for y in w]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for y in w:
        y.main_grad.zero_()
    graph.replay(), graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y.main_grad, 2 * g) for y, g in zip(w, once))
