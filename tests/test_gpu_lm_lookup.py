"""What the LM's token lookup leaves to the module itself, as before there was a lookup of the framework's own."""
import pytest
import torch
import torch.nn as nn

from hdcmamba_b200 import training
from hdcmamba_b200.lm import embed

pytestmark = pytest.mark.gpu


def table(**kw):
    torch.manual_seed(0)
    return nn.Embedding(20, 16, **kw).cuda()


IDS = [[3, 1, 3], [7, 0, 19]]


class Lookup(nn.Module):
    def __init__(self, m):
        super().__init__()
        self.m = m

    def forward(self, ids):
        return embed(self.m, ids)


def test_modules_of_other_kinds():
    class Sum(nn.Module):
        def __init__(self):
            super().__init__()
            self.parts = nn.ModuleList([table(), table()])

        def forward(self, ids):
            return self.parts[0](ids) + self.parts[1](ids)

    ids = torch.tensor(IDS).cuda()
    m = Sum()
    assert torch.equal(embed(m, ids), m(ids))
    f = table().weight.detach()
    assert torch.equal(embed(lambda i: f[i], ids), f[ids])


def test_hooks_of_every_kind_are_called():
    """Forward and backward hooks of the module, and those that are registered for all modules."""
    ids = torch.tensor(IDS).cuda()
    for name in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"):
        for owner in ("module", "all"):
            m, called = table(), []
            if owner == "module":
                handle = getattr(m, name)(lambda *a: called.append(1))
            else:
                name_all = name.replace("register_", "register_module_")
                if not hasattr(nn.modules.module, name_all):
                    continue
                handle = getattr(nn.modules.module, name_all)(lambda *a: called.append(1))
            embed(m, ids).sum().backward()
            handle.remove()
            assert called, (name, owner)


def test_a_forward_of_the_instance_or_of_the_class():
    ids = torch.tensor(IDS).cuda()
    m = table()
    m.forward = lambda i: nn.functional.embedding(i, m.weight) + 1
    assert torch.equal(embed(m, ids), m.weight[ids] + 1)
    m, was = table(), nn.Embedding.forward
    try:
        nn.Embedding.forward = lambda self, i: was(self, i) + 2
        assert torch.equal(embed(m, ids), m.weight[ids] + 2)
    finally:
        nn.Embedding.forward = was


def test_modes_see_the_lookup():
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode
    ids, m, seen = torch.tensor(IDS).cuda(), table(), []

    class Functions(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(getattr(func, "__name__", ""))
            return func(*args, **(kwargs or {}))

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    for mode in (Functions, Dispatch):
        seen.clear()
        with mode():
            y = embed(m, ids)
        assert torch.equal(y, m.weight[ids]) and any("embedding" in s for s in seen), (mode, seen)


def test_tables_that_the_kernel_does_not_take():
    """Rows whose elements lie apart, rows wider than the kernel's, host tables."""
    ids = torch.tensor(IDS).cuda()
    m = table()
    m.weight = nn.Parameter(m.weight.detach().t().contiguous().t())
    assert torch.equal(embed(m, ids), m.weight[ids])
    embed(m, ids).sum().backward()
    want = torch.zeros(20, 16, device="cuda").index_add_(0, ids.flatten(), torch.ones(6, 16, device="cuda"))
    assert torch.equal(m.weight.grad, want)
    m = nn.Embedding(3, 65537, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(embed(m, ids % 3), m.weight[ids % 3])
    m = nn.Embedding(20, 16)
    assert torch.equal(embed(m, ids.cpu()), m.weight[ids.cpu()])
    with pytest.raises(RuntimeError):
        embed(table(), ids.float())


@pytest.mark.parametrize("padding_idx", [None, 3])
def test_gradients_of_the_gradients(padding_idx):
    """The lookup is linear in its table: as with the module, derivatives of every order."""
    ids = torch.tensor(IDS).cuda()
    m = table(padding_idx=padding_idx)
    m.weight.data.normal_()

    def chain(look):
        w = m.weight
        (g,) = torch.autograd.grad((look(m, ids) ** 3).sum(), [w], create_graph=True)
        (h,) = torch.autograd.grad((g ** 2).sum(), [w], create_graph=True)
        (t,) = torch.autograd.grad((h * torch.arange(16, device="cuda")).sum(), [w])
        return g, h, t

    for a, b in zip(chain(embed), chain(lambda mod, i: mod(i))):
        assert (a - b).abs().max() <= 2.0 ** -24 * 64 * b.abs().max()  # some ten products and sums of up to four terms


def test_gradients_of_the_scaled_lookup_against_differences():
    ids = torch.tensor(IDS).cuda()
    w = torch.randn(20, 16, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    u, v = (torch.randn(s, generator=torch.Generator().manual_seed(2)).cuda() for s in ((2, 3, 16), (20, 16)))
    dy = u.clone().requires_grad_()
    (g,) = torch.autograd.grad(training.embedding(ids, w, scale=1.5, padding_idx=1), [w], dy, create_graph=True)
    (d,) = torch.autograd.grad(g, [dy], v)
    want = 1.5 * v[ids] * (ids != 1)[..., None]
    assert torch.equal(d, want)


def test_tangents_and_transforms():
    """Forward-mode derivatives and torch.func's transforms go through the module."""
    import torch.autograd.forward_ad as fwd
    ids, m = torch.tensor(IDS).cuda(), table()
    t = torch.randn_like(m.weight)
    with fwd.dual_level():
        w = fwd.make_dual(m.weight.detach(), t)
        del m._parameters["weight"]
        m.weight = w
        assert torch.equal(fwd.unpack_dual(embed(m, ids)).tangent, t[ids])
    m = table()

    def loss(w):
        y = torch.func.functional_call(Lookup(m), {"m.weight": w}, (ids,))
        return (y ** 2).sum()

    g = torch.func.grad(loss)(m.weight.detach())
    want = torch.zeros_like(g).index_add_(0, ids.flatten(), 2 * m.weight.detach()[ids.flatten()])
    assert (g - want).abs().max() <= 2.0 ** -22 * want.abs().max()
    many = torch.stack([m.weight.detach(), 2 * m.weight.detach()])
    assert torch.equal(torch.vmap(lambda w: torch.func.functional_call(Lookup(m), {"m.weight": w}, (ids,)))(many), many[:, ids])


def test_tensor_subclasses_see_the_lookup():
    seen = []

    class Watched(torch.Tensor):
        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            seen.append(getattr(func, "__name__", ""))
            return super().__torch_function__(func, types, args, kwargs or {})

    ids, m = torch.tensor(IDS).cuda(), table()
    for which in ("ids", "weight"):
        seen.clear()
        if which == "weight":
            w = m.weight.detach().as_subclass(Watched)
            del m._parameters["weight"]
            m.weight = w
        y = embed(m, ids.as_subclass(Watched) if which == "ids" else ids)
        assert isinstance(y, Watched) and "embedding" in seen, (which, seen)


@pytest.mark.parametrize("padding_idx", [None, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_batched_gradients(padding_idx, dtype):
    """Several gradients at once (is_grads_batched), as the module gives them."""
    ids = torch.tensor(IDS).cuda()
    m = table(padding_idx=padding_idx).to(dtype)
    dy = torch.randn(4, 2, 3, 16, generator=torch.Generator().manual_seed(1)).cuda().to(dtype)
    one = [torch.autograd.grad(embed(m, ids), [m.weight], d)[0] for d in dy]
    (got,) = torch.autograd.grad(embed(m, ids), [m.weight], dy, is_grads_batched=True)
    tol = 2 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23  # sums of two terms, rounded once
    assert (got - torch.stack(one)).abs().max() <= tol * got.abs().max()
    # the gradient's own gradient, batched
    y = dy[0].clone().requires_grad_()
    (g,) = torch.autograd.grad(embed(m, ids), [m.weight], y, create_graph=True)
    v = torch.randn(3, 20, 16, generator=torch.Generator().manual_seed(2)).cuda().to(dtype)
    (d,) = torch.autograd.grad(g, [y], v, is_grads_batched=True)
    want = v[:, ids] * (1 if padding_idx is None else (ids != padding_idx)[..., None])
    assert torch.equal(d, want)
