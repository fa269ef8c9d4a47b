"""What the operators' autograd nodes refuse beside bad arguments, checked without a GPU (the checks come before anything
touches a device): tracers, which would record a result's allocation and not the kernel that fills it, function
transforms and tensors without memory.  The public functions are under the same tests on a GPU in test_gpu_tracing.py."""
import pytest
import torch

from unicorn_amd import native

X = torch.randn(4, 8)
TEACHER, INDEX = torch.randn(4, 3), torch.zeros(4, 3, dtype=torch.int64)
NODES = {"layer_norm": lambda x: native.nodes().layer_norm(x, None, None, 1e-5),
         "route": lambda x: native.nodes().route(x, None, 2, 0, 1, 1, 0, True, 1.0)[0],
         "distill": lambda x: native.nodes().distill(x, TEACHER, INDEX, 1.0, 2)}


@pytest.mark.parametrize("name", list(NODES))
def test_tracing_is_refused(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    op = NODES[name]
    with pytest.raises(RuntimeError, match="tracing is not supported"):
        torch.jit.trace(op, (X,))
    with pytest.raises(RuntimeError, match="tracing is not supported"):
        make_fx(op)(X)
    with FakeTensorMode() as mode:
        fake = mode.from_tensor(X)
        with pytest.raises(RuntimeError, match="tracing is not supported"):
            op(fake)
    with pytest.raises(RuntimeError, match="not supported by this operator"):
        op(fake)


@pytest.mark.parametrize("name", list(NODES))
def test_function_transforms_are_refused(name):
    op = NODES[name]
    with pytest.raises(RuntimeError, match="function transforms"):
        torch.func.grad(lambda v: op(v).sum())(X)
    with pytest.raises(RuntimeError, match="function transforms"):
        torch.vmap(op)(X[None])
    with pytest.raises(RuntimeError, match="not supported by this operator"):
        torch.func.functionalize(op)(X)
