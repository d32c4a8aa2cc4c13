"""The 8-bit operators beside autograd: there is no backward, so what would lose a
gradient is refused, and what a call writes is seen to have changed."""
import pytest
import torch

from defer_amd import q8


def calls(t):
    """Every call, with t(shape) for each tensor of values or scales."""
    c = torch.zeros(2, 64, dtype=torch.int8)
    n = torch.ones(2, dtype=torch.int32)
    i = torch.zeros(2, 1, dtype=torch.int32)
    pages = q8.Pages(torch.zeros(2, 1, 64, 64, dtype=torch.int8), torch.zeros(2, 1, 64, 64, dtype=torch.int8),
                     t(2, 1, 64), torch.zeros(2, 1, 64), i)
    x = torch.zeros(2, 64)
    return {
        "quantize": lambda: q8.quantize(t(2, 64)),
        "rms_norm": lambda: q8.rms_norm(t(2, 64), x[0], 1e-5),
        "linear": lambda: q8.linear(c, t(2), c, x[:, 0]),
        "kv_write": lambda: q8.kv_write(pages, t(2, 1, 64), t(2, 1, 64), n),
        "kv_read": lambda: q8.kv_read(pages, n, None, 2, 64),
        "attention": lambda: q8.attention(t(2, 1, 64), pages, n),
    }


@pytest.mark.parametrize("name", ["quantize", "rms_norm", "kv_write", "attention"])
def test_what_requires_a_gradient_is_refused(name):
    call = calls(lambda *s: torch.zeros(*s, requires_grad=True))[name]
    with pytest.raises(ValueError, match="requires a gradient"):
        call()
    with torch.no_grad(), pytest.raises(ValueError, match="not a tensor on a GPU"):  # goes on to the next check
        call()


@pytest.mark.parametrize("name", ["quantize", "rms_norm", "linear", "kv_write", "attention"])
def test_a_trace_is_refused(name):
    def traced(x):
        calls(lambda *s: torch.zeros(*s))[name]()
        return x + 1

    with pytest.raises(ValueError, match="trace"):
        torch.jit.trace(traced, torch.zeros(1), check_trace=False)
    with pytest.raises(ValueError, match="not a tensor on a GPU"):  # and not for ever
        traced(torch.zeros(1))


DEV = "cuda:0"


def cache():
    return q8.new_pages(2, 1, 64, torch.arange(2, dtype=torch.int32, device=DEV)[None])


@pytest.mark.gpu
def test_every_input_that_requires_a_gradient_is_refused():
    x, w = torch.randn(3, 64, device=DEV), torch.ones(64, device=DEV)
    k = x[:, None].contiguous()
    n, start = torch.tensor([3], dtype=torch.int32, device=DEV), torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    c, s = q8.quantize(x)
    p = cache()
    q8.kv_write(p, k, k, n, start)

    def grad(t):
        return t.detach().clone().requires_grad_()

    with_grad = {
        "x": lambda: q8.rms_norm(grad(x), w, 1e-5, residual=x), "weight": lambda: q8.rms_norm(x, grad(w), 1e-5),
        "residual": lambda: q8.rms_norm(x, w, 1e-5, residual=grad(x)), "out": lambda: q8.rms_norm(x, w, 1e-5, residual=x, out=grad(x)),
        "x_scale": lambda: q8.linear(c, grad(s), c, s), "w_scale": lambda: q8.linear(c, s, c, grad(s)),
        "k": lambda: q8.kv_write(p, grad(k), k, n, start), "v": lambda: q8.kv_write(p, k, grad(k), n, start),
        "value_scale": lambda: q8.kv_read(p._replace(value_scale=grad(p.value_scale)), n, start, 3, 64),
        "q": lambda: q8.attention(grad(k), p, n, start), "attention's out": lambda: q8.attention(k, p, n, start, out=grad(k)),
    }
    for name, call in with_grad.items():
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()
    y = q8.linear(c, s, c, s)
    assert not y.requires_grad


@pytest.mark.gpu
def test_what_a_call_writes_has_changed_for_autograd():
    x, r, w = (torch.randn(3, 64, device=DEV) for _ in range(3))
    n, start = torch.tensor([3], dtype=torch.int32, device=DEV), torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    p = cache()
    k = x[:, None].clone()  # apart from x, whose views change with it
    out = torch.empty_like(k)
    writes = {
        "rms_norm": ([x], lambda: q8.rms_norm(x, w[0].contiguous(), 1e-5, residual=r, out=x)),
        "kv_write": (list(p[:4]), lambda: q8.kv_write(p, k, k, n, start)),
        "attention": ([out], lambda: q8.attention(k, p, n, start, out=out)),
    }
    for name, (tensors, call) in writes.items():
        before = [t._version for t in tensors]
        call()
        assert all(t._version > b for t, b in zip(tensors, before)), name
    reads = [r, k, n, p.table]
    before = [t._version for t in reads]
    for _, call in writes.values():
        call()
    assert [t._version for t in reads] == before
    # a tensor that a graph has saved
    a = torch.randn(3, 64, device=DEV, requires_grad=True)
    saved = torch.randn(3, 64, device=DEV)
    y = (a * saved).sum()
    q8.rms_norm(saved, w[0].contiguous(), 1e-5, residual=r, out=saved)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        z = torch.zeros(3, 64, device=DEV)
    q8.rms_norm(x, w[0].contiguous(), 1e-5, residual=r, out=z)  # has no version
    assert torch.equal(z, x + r)
