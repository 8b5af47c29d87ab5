"""The layers as torch.ops.ppo_amd.* on the GPU: opcheck (schema, fake tensor,
autograd registration), the functions' bits, and a compiled layer with its
backward pass.  (A file of its own, as test_gpu_torch_ops.py: torch.compile
switches off the argument validation of torch.distributions for the process.)"""

import pytest
import torch

import ppo_amd

pytestmark = pytest.mark.gpu


def _case(dev, M):
    g = torch.Generator().manual_seed(M)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    D, F = 24, 36
    leaves = [rn(M, D), rn(F, D) * D ** -0.5, rn(F, D) * D ** -0.5, rn(F) * 0.1, rn(F) * 0.1]
    return [t.to(dev).requires_grad_() for t in leaves], rn(M, F).to(dev) * 0.1


def test_registered_operators(dev):
    """opcheck on each operator, and the functions' bits."""
    op = torch.ops.ppo_amd
    leaves, dh = _case(dev, 20)
    rows, seed = torch.arange(20, device=dev) * 3, torch.tensor([4], device=dev)
    utils = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(op.dropout, (leaves[0], 0.3, 4, None, rows), test_utils=utils)
    torch.library.opcheck(op.gated_ffn, (*leaves, "silu", 0.2, 0, seed, rows), test_utils=utils)
    plain = [v.detach() for v in leaves]
    torch.library.opcheck(op.quantize_rows, (plain[0],), test_utils=utils)
    q, s = ppo_amd.quantize_rows(plain[1])
    torch.library.opcheck(op.int8_linear, (plain[0], q, s, None, None, None), test_utils=utils)

    h, _ = op.gated_ffn(*leaves, "silu", 0.2, 0, seed, rows)
    z = op.dropout(h, 0.1, 4, None, rows)
    got = [z.detach(), *torch.autograd.grad(z, leaves, dh)]
    h = ppo_amd.gated_ffn(*leaves, dropout_p=0.2, seed=seed, rows=rows)
    z = ppo_amd.dropout(h, 0.1, 4, rows)
    want = [z.detach(), *torch.autograd.grad(z, leaves, dh)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_registered_backward_refuses(dev):
    """The registered backward pass checks its arguments as the functions do."""
    leaves, dh = _case(dev, 20)
    x, wg, wu = (t.detach() for t in leaves[:3])
    saved = torch.randn(2, 20, 36, device=dev)
    f = torch.ops.ppo_amd.gated_ffn_backward

    def call(dh=dh, x=x, wg=wg, wu=wu, saved=saved, seed_at=None, rows=None):
        return f(dh, x, wg, wu, saved, True, "silu", 0.1, 1, seed_at, rows)

    assert [tuple(t.shape) for t in call()] == [(20, 24), (36, 24), (36, 24), (36,), (36,)]
    for kw in (dict(dh=dh[:19].contiguous()), dict(saved=saved[:, :19].contiguous()),
               dict(dh=dh.t().contiguous().t()), dict(wu=wu[:35].contiguous()),
               dict(rows=torch.arange(19, device=dev)), dict(seed_at=torch.arange(2, device=dev))):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(dh=dh.half()), dict(saved=saved.half()),
               dict(rows=torch.arange(20, device=dev, dtype=torch.int32))):
        with pytest.raises(TypeError):
            call(**kw)
    for kw in (dict(saved=saved.cpu()), dict(rows=torch.arange(20)),
               dict(seed_at=torch.tensor([1]))):
        with pytest.raises(RuntimeError, match="no CPU fallback|expected"):
            call(**kw)


def test_registered_operators_compile(dev):
    """A compiled layer with its backward is traced whole and equals eager."""
    op = torch.ops.ppo_amd
    leaves, dh = _case(dev, 40)

    def layer(x, wg, wu, bg, bu, seed):
        h = op.gated_ffn(x, wg, wu, bg, bu, "gelu", 0.2, 0, seed, None)[0]
        return op.dropout(h, 0.1, 0, seed, None) * 2.0

    compiled = torch.compile(layer, fullgraph=True, backend="aot_eager")
    for k in (3, 9):
        seed = torch.tensor([k], device=dev)
        runs = []
        for f in (layer, compiled):
            y = f(*leaves, seed)
            runs.append([y.detach(), *torch.autograd.grad(y, leaves, dh)])
        assert all(torch.equal(a, b) for a, b in zip(*runs))
