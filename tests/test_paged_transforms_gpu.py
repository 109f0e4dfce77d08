"""GPU: what records, transforms or differentiates a program sees the paged cache's operators, although their usual calls
go past the dispatcher: tracing, dispatch modes, tangents, function transforms, negative views, tensor subclasses."""
import pytest
import torch
from torch.autograd import forward_ad

from intrasm_engine_b200.pytorch import paged_attention as paged

from . import paged_util as U
from .paged_util import DEV

pytestmark = pytest.mark.gpu

LENGTHS, HEADS, KV, DIM, PAGE = [70, 33, 0], 4, 2, 64, 16


def operands():
    """name -> (function of all operands, the operands' names), and the operands."""
    gen = torch.Generator().manual_seed(3)
    k_cache, v_cache, table = U.make_cache(gen, LENGTHS, KV, DIM, PAGE, torch.float16, fill=0.0)
    cos, sin = paged.rope_table(80, DIM, device=DEV)
    x = dict(k_cache=k_cache, v_cache=v_cache, cos=cos, sin=sin, boxes=U.boxes_of(k_cache, table, LENGTHS, PAGE))
    for name, heads in (("q", HEADS), ("k", KV), ("v", KV)):
        x[name] = torch.randn(len(LENGTHS), heads, DIM, generator=gen).half().to(DEV)
    held = torch.tensor(LENGTHS, dtype=torch.int32, device=DEV)
    calls = {
        "append": (lambda q, k, v, k_cache, v_cache, cos, sin, boxes: paged.paged_append(
            q, k, v, k_cache, v_cache, table, held, rope=(cos, sin), boxes=boxes),
                   ("q", "k", "v", "k_cache", "v_cache", "cos", "sin", "boxes")),
        "attention": (lambda q, k_cache, v_cache: paged.paged_attention(q, k_cache, v_cache, table, held),
                      ("q", "k_cache", "v_cache")),
        "select": (lambda q, boxes: paged.paged_select(q, boxes, table, held, PAGE, 3), ("q", "boxes")),
    }
    return calls, x


@pytest.fixture(params=["append", "attention", "select"])
def call(request):
    """A function, its operands, and which of them may be looked at one by one."""
    calls, x = operands()
    f, names = calls[request.param]
    return f, [x[n].clone() for n in names], names


def test_tangents_are_not_dropped(call):
    f, args, names = call
    for i, name in enumerate(names):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]
            with pytest.raises(NotImplementedError, match=name):
                f(*dual)
    f(*args)


def test_forward_transform_is_refused(call):
    f, args, names = call
    for i, name in enumerate(names):
        with pytest.raises(NotImplementedError, match=name):
            torch.func.jvp(lambda a: f(*args[:i], a, *args[i + 1:]).float(), (args[i],), (torch.ones_like(args[i]),))


def test_backward_transform_is_refused(call):
    f, args, names = call
    for i, name in enumerate(names):
        with pytest.raises(RuntimeError, match=name + " requires a gradient"):
            torch.func.grad(lambda a: f(*args[:i], a, *args[i + 1:]).float().sum())(args[i])


def test_operands_that_require_a_gradient(call):
    """Refused, also through the dispatcher; without gradients they are tensors like others."""
    f, args, names = call
    ref = f(*[a.clone() for a in args])
    wanted = args[0].clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match=names[0] + " requires a gradient"):
        f(wanted, *args[1:])
    with pytest.raises(RuntimeError, match=names[0] + " requires a gradient"):
        f(torch._neg_view(wanted), *args[1:])
    with torch.no_grad():
        assert torch.equal(f(wanted, *args[1:]), ref)
    with torch.inference_mode():
        assert torch.equal(f(*[a.clone() for a in args]), ref)


def test_trace_follows_the_input(call):
    f, args, _ = call
    traced = torch.jit.trace(f, tuple(a.clone() for a in args), check_trace=False)
    other = [torch.randn_like(args[0])] + args[1:]
    assert torch.equal(traced(*[a.clone() for a in other]), f(*[a.clone() for a in other]))


def test_dispatch_mode_sees_the_operators(call):
    from torch.fx.experimental.proxy_tensor import make_fx
    f, args, _ = call
    graph = make_fx(f)(*[a.clone() for a in args])
    assert any("iex_ops.paged" in str(node.target) for node in graph.graph.nodes)
    other = [torch.randn_like(args[0])] + args[1:]
    assert torch.equal(graph(*[a.clone() for a in other]), f(*[a.clone() for a in other]))


def test_vmap_gives_the_same_or_is_refused(call):
    """Over queries: the operators that write nothing run one by one, appending is refused."""
    f, args, names = call
    both = torch.stack([args[0], -args[0]])
    if "k" in names:
        with pytest.raises(RuntimeError):
            torch.vmap(lambda q: f(q, *args[1:]))(both)
    else:
        assert torch.equal(torch.vmap(lambda q: f(q, *args[1:]))(both), torch.stack([f(q, *args[1:]) for q in both]))


def test_negative_view(call):
    """A query that only says it is negated."""
    f, args, _ = call
    assert torch.equal(f(torch._neg_view(args[0]), *[a.clone() for a in args[1:]]),
                       f(-args[0], *[a.clone() for a in args[1:]]))


def test_subclass_reaches_its_own_dispatch(call):
    class Wrapped(torch.Tensor):
        @staticmethod
        def __new__(cls, inner):
            return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

        def __init__(self, inner):
            self.inner = inner

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            seen.append(str(func))
            unwrap = lambda t: t.inner if isinstance(t, cls) else t
            return func(*(unwrap(a) for a in args), **(kwargs or {}))

    f, args, _ = call
    seen = []
    out = f(Wrapped(args[0]), *[a.clone() for a in args[1:]])
    assert seen and torch.equal(out, f(*[a.clone() for a in args]))
