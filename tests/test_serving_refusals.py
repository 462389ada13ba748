"""What linear() and moe_few_tokens() refuse: shapes, types and strides are checked before the device, so no GPU is needed."""

import pytest
import torch

from revealaiccl_b200.ops import _native

if not _native.has_kernels():  # pragma: no cover
    pytest.skip("kernel library not built", allow_module_level=True)

BF16 = torch.bfloat16


def _linear(**kw):
    from revealaiccl_b200.ops.linear import linear
    a = dict(x=torch.zeros(3, 16, dtype=BF16), weight=torch.zeros(8, 16, dtype=BF16))
    a.update(kw)
    return linear(a.pop("x"), a.pop("weight"), a.pop("bias", None), **a)


def _moe(**kw):
    from revealaiccl_b200.ops.moe_few import moe_few_tokens
    a = dict(x=torch.zeros(3, 16, dtype=BF16), router_w=torch.zeros(4, 16, dtype=BF16), w1=torch.zeros(4, 24, 16, dtype=BF16),
             w2=torch.zeros(4, 10, 12, dtype=BF16), top_k=2)
    a.update(kw)
    return moe_few_tokens(**a)


X = torch.zeros(3, 16, dtype=BF16)


@pytest.mark.parametrize("kw,words", [
    (dict(), "CUDA device"),
    (dict(act="tanh"), "act must be one of"),
    (dict(x=torch.zeros(16, dtype=BF16)), r"x is \[M, K\]"),
    (dict(weight=torch.zeros(8, 15, dtype=BF16)), "15 columns"),
    (dict(weight=torch.zeros(7, 16, dtype=BF16), act="swiglu"), "as many up rows"),
    (dict(weight=torch.zeros(8, 16)), "both be bf16 or both be fp32"),
    (dict(x=X.half(), weight=torch.zeros(8, 16).half()), "both be bf16 or both be fp32"),
    (dict(x=torch.zeros(16, 3, dtype=BF16).t()), "contiguous rows"),
    (dict(bias=torch.zeros(8, dtype=BF16)), "bias must be a contiguous fp32"),
    (dict(bias=torch.zeros(7)), "bias must be a contiguous fp32"),
    (dict(residual=torch.zeros(3, 7)), "shape of the output"),
    (dict(residual=torch.zeros(8, 3).t()), "residual must be fp32 or bf16 with contiguous rows"),
    (dict(out=torch.zeros(2, 8, dtype=BF16)), "out must have shape"),
    (dict(out=torch.zeros(3, 8), out_dtype=BF16), "another type"),
    (dict(out=torch.zeros(8, dtype=BF16).expand(3, 8)), "do not overlap"),
    (dict(out_dtype=torch.float16), "the output is fp32"),
    (dict(x=X.float(), weight=torch.zeros(8, 16), out_dtype=BF16), "the output is fp32"),
    (dict(x=torch.zeros(2 ** 21 + 1, 0, dtype=BF16), weight=torch.zeros(8, 0, dtype=BF16)), r"at most 2\^21 rows"),
])
def test_linear_refuses(kw, words):
    with pytest.raises(ValueError, match=words):
        _linear(**kw)


@pytest.mark.parametrize("kw,words", [
    (dict(), "CUDA device"),
    (dict(act="tanh"), "act must be one of"),
    (dict(gate_mode="sigmoid"), "gate_mode must be one of"),
    (dict(x=torch.zeros(65, 16, dtype=BF16)), "at most 64 tokens"),
    (dict(router_w=torch.zeros(256, 16, dtype=BF16)), "1 to 255 experts"),
    (dict(router_w=torch.zeros(0, 16, dtype=BF16)), "1 to 255 experts"),
    (dict(top_k=0), "top_k"),
    (dict(top_k=5), "top_k"),
    (dict(w1=torch.zeros(4, 12, 16, dtype=BF16)), "shapes differ"),
    (dict(w2=torch.zeros(3, 10, 12, dtype=BF16)), "shapes differ"),
    (dict(w1=torch.zeros(4, 24, 15, dtype=BF16)), "shapes differ"),
    (dict(w2=torch.zeros(4, 10, 0, dtype=BF16), w1=torch.zeros(4, 0, 16, dtype=BF16)), "widths"),
    (dict(w1=torch.zeros(4, 24, 16)), "all be bf16 or all be fp32"),
    (dict(w1=torch.zeros(4, 16, 24, dtype=BF16).transpose(1, 2)), "contiguous rows"),
    (dict(router_b=torch.zeros(3)), "router_b"),
    (dict(b1=torch.zeros(4, 12)), "b1"),
    (dict(b2=torch.zeros(4, 10, dtype=BF16)), "b2"),
    (dict(block_mask=torch.zeros(4)), "block_mask"),
    (dict(block_mask=torch.zeros(2, 4, dtype=torch.bool)), "block_mask"),
    (dict(residual=torch.zeros(3, 12)), "shape of the output"),
    (dict(out=torch.zeros(3, 11)), "out must have shape"),
])
def test_moe_refuses(kw, words):
    with pytest.raises(ValueError, match=words):
        _moe(**kw)


def test_gradients_are_refused():
    with pytest.raises(RuntimeError, match="no backward"):
        _linear(weight=torch.zeros(8, 16, requires_grad=True), x=torch.zeros(3, 16))
    with pytest.raises(RuntimeError, match="no backward"):
        _moe(w2=torch.zeros(4, 10, 12, dtype=BF16, requires_grad=True))
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
        _linear(weight=torch.zeros(8, 16, requires_grad=True), x=torch.zeros(3, 16))


def test_shared_memory_is_refused():
    buf = torch.zeros(3, 24, dtype=BF16)
    with pytest.raises(ValueError, match="shares memory with an input"):
        _linear(x=buf[:, :16], out=buf[:, 16:])
    r = torch.zeros(4, 8, dtype=BF16)
    with pytest.raises(ValueError, match="shares memory with residual"):
        _linear(residual=r[:3], out=r[1:])
    with pytest.raises(ValueError, match="CUDA device"):
        _linear(residual=r[:3], out=r[:3])


def test_out_apart_from_biases_and_mask():
    buf = torch.zeros(64)
    with pytest.raises(ValueError, match="shares memory with an input"):
        _linear(bias=buf[4:12], out=buf[:24].view(3, 8), out_dtype=torch.float32)
    with pytest.raises(ValueError, match="shares memory with an input"):
        _moe(router_b=buf[28:32], out=buf[:30].view(3, 10), out_dtype=torch.float32)


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        x = fwd.make_dual(torch.zeros(3, 16), torch.ones(3, 16))
        with pytest.raises(RuntimeError, match="no derivative"):
            _linear(x=x, weight=torch.zeros(8, 16))
        with torch.no_grad(), pytest.raises(RuntimeError, match="no derivative"):
            _linear(x=x, weight=torch.zeros(8, 16))
        with pytest.raises(RuntimeError, match="no derivative"):
            _linear(weight=torch.zeros(8, 16), x=torch.zeros(3, 16), residual=fwd.make_dual(torch.zeros(3, 8), torch.ones(3, 8)))
        w2 = torch.zeros(4, 10, 12)
        with pytest.raises(RuntimeError, match="no derivative"):
            _moe(x=torch.zeros(3, 16), router_w=torch.zeros(4, 16), w1=torch.zeros(4, 24, 16), w2=fwd.make_dual(w2, w2 + 1))
        with pytest.raises(ValueError, match="CUDA device"):
            _linear(x=fwd.unpack_dual(x).primal, weight=torch.zeros(8, 16))


def _freed(*shape, dtype=BF16):
    t = torch.zeros(*shape, dtype=dtype)
    t.untyped_storage().resize_(0)
    return t


@pytest.mark.parametrize("t", [_freed(3, 16), torch.zeros(3, 16, dtype=BF16).to_sparse(), torch._neg_view(torch.zeros(3, 16, dtype=BF16)),
                               torch._efficientzerotensor((3, 16), dtype=BF16)], ids=["freed", "sparse", "neg", "zero"])
def test_tensors_without_their_numbers_are_refused(t):
    with pytest.raises(ValueError, match="x (reaches behind its storage|must be a dense tensor)"):
        _linear(x=t)
    with pytest.raises(ValueError, match="x (reaches behind its storage|must be a dense tensor)"):
        _moe(x=t)


def test_freed_storages_are_refused():
    for name, shape, dtype in (("weight", (8, 16), BF16), ("bias", (8,), torch.float32), ("residual", (3, 8), BF16), ("out", (3, 8), BF16)):
        with pytest.raises(ValueError, match=f"{name} reaches behind its storage"):
            _linear(**{name: _freed(*shape, dtype=dtype)})
    for name, shape, dtype in (("router_w", (4, 16), BF16), ("w1", (4, 24, 16), BF16), ("w2", (4, 10, 12), BF16),
                               ("router_b", (4,), torch.float32), ("b1", (4, 24), torch.float32), ("b2", (4, 10), torch.float32),
                               ("block_mask", (3, 4), torch.bool), ("residual", (3, 10), BF16), ("out", (3, 10), BF16)):
        with pytest.raises(ValueError, match=f"{name} reaches behind its storage"):
            _moe(**{name: _freed(*shape, dtype=dtype)})
    part = torch.zeros(6, 16, dtype=BF16)[3:]
    part.untyped_storage().resize_(100)
    with pytest.raises(ValueError, match="x reaches behind its storage, which holds 100 bytes"):
        _linear(x=part)


class _Wrapper(torch.Tensor):
    """A shape without memory, as distributed and quantised tensors are."""

    @staticmethod
    def __new__(cls, *shape, dtype=BF16):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(func)


def test_wrappers_are_refused():
    for name, shape in (("x", (3, 16)), ("weight", (8, 16)), ("residual", (3, 8)), ("out", (3, 8))):
        with pytest.raises(ValueError, match=f"{name} has no memory"):
            _linear(**{name: _Wrapper(*shape)})
    for name, shape in (("x", (3, 16)), ("router_w", (4, 16)), ("w1", (4, 24, 16)), ("w2", (4, 10, 12)), ("residual", (3, 10)),
                        ("out", (3, 10))):
        with pytest.raises(ValueError, match=f"{name} has no memory"):
            _moe(**{name: _Wrapper(*shape)})
    with pytest.raises(ValueError, match="b1 has no memory"):
        _moe(b1=_Wrapper(4, 24, dtype=torch.float32))
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        fake = torch.zeros(3, 16, dtype=BF16)
    with pytest.raises((ValueError, RuntimeError), match="memory|data pointer"):
        _linear(x=fake)
    with pytest.raises(ValueError, match="CUDA device"):
        _linear(x=torch.zeros(3, 16, dtype=BF16, device="meta"), weight=torch.zeros(8, 16, dtype=BF16, device="meta"))
