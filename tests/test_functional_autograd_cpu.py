"""CPU: what the autograd functions of ivid_amd.functional hand to the library, with the launch itself replaced.  The library's host
code (scratch sizes, refusals) is the real one; tensors live on the CPU and only the stand-in below touches them."""
import ctypes
import threading

import pytest
import torch

SIZES = {0: 4, 1: 2, 2: 2}      # bytes of an element by the library's dtype code


@pytest.fixture
def host(monkeypatch):
    """ivid_amd.functional over CPU tensors.  `launches` collects (name, arguments), a descriptor
    as it was then; a dropout with p = 0 copies, another zeroes."""
    from ivid_amd import _lib, functional as F

    def launch(name, device, *args):
        if name.startswith("ivid_gn_act"):
            args = (_lib.GnActDesc.from_buffer_copy(args[0]._obj),) + args[1:]
        F.launches.append((name, args))
        if name == "ivid_dropout":
            dtype, src, dst, n, p = args[:5]
            if p == 0:
                ctypes.memmove(dst, src, n * SIZES[dtype])
            else:
                ctypes.memset(dst, 0, n * SIZES[dtype])
    monkeypatch.setattr(F, "launches", [], raising=False)
    monkeypatch.setattr(F, "_check_x", lambda x, name: None)
    monkeypatch.setattr(F, "_launch", launch)
    monkeypatch.setattr(F, "_refuse_capture", lambda: None)
    return F


@pytest.mark.parametrize("rng", [None, (1, 2), "tensor"])
@pytest.mark.parametrize("shape", [(7, 3), (0, 3)], ids=["full", "empty"])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_dropout_has_a_gradient_with_every_form_of_rng(host, p, shape, rng):
    """p = 0 draws nothing and needs no rng, in the backward pass either; nor has an empty tensor anything to draw."""
    if rng is None and p > 0 and shape[0]:
        pytest.skip("p > 0 needs rng")
    if rng == "tensor":
        rng = torch.tensor([1, 2])
    x = torch.randn(shape).requires_grad_()
    dy = torch.randn(shape)
    for create_graph in (False, True):
        y = host.dropout(x, p, rng) if rng is not None else host.dropout(x, p)
        (dx,) = torch.autograd.grad(y, x, dy, create_graph=create_graph)
        assert torch.equal(dx, dy if p == 0 else torch.zeros_like(dy))
    for name, args in host.launches:
        assert args[4] == p and args[5:] == ((1, 2, None) if isinstance(rng, tuple) and p else (0, 0, rng.data_ptr() if p else None))


def _norm_inputs(n=2, hw=6, c=8, spread=1):
    """x (strided with spread > 1, so that the backward pass describes it anew), weight, bias; all leaves"""
    x = torch.randn(n, hw, c * spread)[..., :c].detach().requires_grad_()
    return x, torch.ones(c).requires_grad_(), torch.zeros(c).requires_grad_()


@pytest.mark.parametrize("spread", [1, 2], ids=["in place", "strided"])
def test_a_rewritten_list_of_seed_and_stream_does_not_reach_the_backward_pass(host, spread):
    """rng may be any pair of integers; what the forward pass drew with is what the gradient is drawn with."""
    rng = [5, 6]
    x, w, b = _norm_inputs(spread=spread)
    a, y = host.dropout(x, 0.25, rng), host.group_norm_act(x, 2, w, b, p=0.25, rng=rng)
    rng[0] = 7
    torch.autograd.grad([a, y], [x, w, b], [torch.ones_like(a), torch.ones_like(y)])
    drawn = {}
    for name, args in host.launches:
        seed = args[5:7] if name == "ivid_dropout" else (args[0].seed, args[0].stream_id)
        drawn.setdefault(name, []).append(seed)
    assert drawn == {"ivid_dropout": [(5, 6)] * 2, "ivid_gn_act_forward": [(5, 6)], "ivid_gn_act_backward": [(5, 6)]}


def test_forward_mode_tangents_are_refused(host):
    """The kernels propagate no tangent: an output without one would read as a zero derivative."""
    import torch.autograd.forward_ad as fwd
    from ivid_amd._lib import IvidHipError
    F = host
    n, hw, c = 2, 6, 8
    t = dict(x=torch.randn(n, hw, c), weight=torch.ones(c), bias=torch.zeros(c), film=torch.zeros(n, 4 * c), skip=torch.randn(n, hw, c))
    t["weight"], t["bias"] = torch.ones(2 * c), torch.zeros(2 * c)
    y, stats = F.group_norm_act_forward(groups=2, **t)
    count = len(F.launches)
    with fwd.dual_level():
        for grad in (True, False):      # with gradients enabled or not, for tensors that ask for none
            with torch.set_grad_enabled(grad):
                with pytest.raises(IvidHipError, match="tangent"):
                    F.dropout(fwd.make_dual(t["x"], torch.ones_like(t["x"])), 0.0)
                for k in t:
                    dual = dict(t, **{k: fwd.make_dual(t[k], torch.ones_like(t[k]))})
                    for fn in (F.group_norm_act, F.group_norm_act_forward, lambda **kw: F.group_norm_act_backward(y, stats, **kw)):
                        with pytest.raises(IvidHipError, match="tangent"):
                            fn(groups=2, **dual)
                for k, v in (("dy", y), ("stats", stats)):
                    args = dict(dict(dy=y, stats=stats), **{k: fwd.make_dual(v, torch.ones_like(v))})
                    with pytest.raises(IvidHipError, match="tangent"):
                        F.group_norm_act_backward(groups=2, **args, **t)
        # a gradient with a tangent, forward over reverse
        x = t["x"].clone().requires_grad_()
        for out in (F.dropout(x, 0.0), F.group_norm_act(x, 2, torch.ones(c), torch.zeros(c))):
            count += 1
            with pytest.raises(IvidHipError, match="tangent"):
                torch.autograd.grad(out, x, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)))
        # tensors without a tangent are as they are elsewhere
        assert F.group_norm_act(groups=2, **t).shape == y.shape and F.dropout(t["x"], 0.0).shape == t["x"].shape
    assert len(F.launches) == count + 2


@pytest.mark.parametrize("spread", [1, 2], ids=["in place", "strided"])
def test_two_threads_walk_one_retained_graph(host, monkeypatch, spread):
    """Each backward pass launches on the tensors that it unpacked itself (here filled with the thread's number), or on its own
    copies of them, and they live until the launch has returned."""
    x, w, b = _norm_inputs(spread=spread)
    me = threading.local()

    def unpack(t):
        return t.clone().fill_(me.number) if spread == 1 else torch.full(t.shape + (2,), float(me.number))[..., 0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = host.group_norm_act(x, 2, w, b)
    both = threading.Barrier(2, timeout=60)
    seen, failed = {}, []

    def launch(name, device, desc, *args):
        both.wait()      # both have described their call
        d = desc._obj
        seen[me.number] = [ctypes.c_float.from_address(q).value for q in (d.src0, d.gamma, d.beta)]
        both.wait()
    monkeypatch.setattr(host, "_launch", launch)

    def walk(number):
        me.number = number
        try:
            with torch.autograd.set_multithreading_enabled(False):
                torch.autograd.grad(y, [x, w, b], torch.ones_like(y), retain_graph=True)
        except Exception as e:      # noqa: BLE001
            failed.append(e)
            both.abort()
    threads = [threading.Thread(target=walk, args=(i,)) for i in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not failed
    assert seen == {i: [float(i)] * 3 for i in (1, 2)}


@pytest.mark.parametrize("spread", [1, 2], ids=["in place", "strided"])
@pytest.mark.parametrize("which", ["x", "skip", "weight", "bias", "film", "stats"])
def test_saved_tensors_that_come_back_as_others_are_refused(host, which, spread):
    """A hook that unpacks another type or shape than it was given: the launch would read past their ends."""
    n, hw, c = 2, 6, 8
    x, _, _ = _norm_inputs(n, hw, c, spread)
    t = dict(x=x, skip=torch.randn(n, hw, c), weight=torch.ones(2 * c), bias=torch.zeros(2 * c), film=torch.zeros(n, 4 * c))
    for bad in (lambda s: s.half(), lambda s: s[:1], lambda s: s.unsqueeze(0)):
        order = []
        with torch.autograd.graph.saved_tensors_hooks(lambda s: (len(order), order.append(1), s)[::2],
                                                      lambda k: bad(k[1]) if k[0] == ["x", "weight", "bias", "film", "skip", "stats"].index(which) else k[1]):
            y = host.group_norm_act(groups=2, **t)
        host.launches.clear()
        with pytest.raises((ValueError, RuntimeError), match="saved|stats"):
            torch.autograd.grad(y, x, torch.ones_like(y))
        assert not host.launches


def test_a_saved_rng_that_comes_back_as_another_is_refused(host):
    x, w, b = _norm_inputs()
    for bad in (lambda s: s.int(), lambda s: s[:1], lambda s: s.to("meta")):
        with torch.autograd.graph.saved_tensors_hooks(lambda s: s, lambda s: bad(s) if s.dtype == torch.int64 else s):
            ys = [host.group_norm_act(x, 2, w, b, p=0.5, rng=torch.tensor([1, 2])), host.dropout(x, 0.5, torch.tensor([1, 2]))]
        host.launches.clear()
        for y in ys:
            with pytest.raises(ValueError, match="rng"):
                torch.autograd.grad(y, x, torch.ones_like(y))
        assert not host.launches


def test_statistics_that_come_back_with_other_strides(host, monkeypatch):
    x, w, b = _norm_inputs(n=3)
    values = torch.arange(12.0).reshape(3, 2, 2)

    def unpack(t):      # the statistics have a shape of their own
        return values.clone().transpose(0, 2).contiguous().transpose(0, 2) if t.shape == values.shape else t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = host.group_norm_act(x, 2, w, b)
    seen = []
    monkeypatch.setattr(host, "_launch", lambda name, device, desc, stats, *args: seen.append(
        [ctypes.c_float.from_address(stats + 4 * i).value for i in range(12)]))
    torch.autograd.grad(y, x, torch.ones_like(y))
    assert seen == [values.reshape(-1).tolist()]


@pytest.mark.parametrize("spread", [1, 2], ids=["in place", "strided"])
def test_a_backward_pass_that_finds_the_call_taken(host, spread):
    """... by another thread describes its own from the saved tensors, to the same launch, and refuses the same."""
    n, hw, c = 2, 6, 8
    x, _, _ = _norm_inputs(n, hw, c, spread)
    t = dict(x=x, skip=torch.randn(n, hw, c), weight=torch.ones(2 * c), bias=torch.zeros(2 * c), film=torch.zeros(n, 4 * c))
    rng = torch.tensor([1, 2])
    swap = [lambda s: s]
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s, lambda s: swap[0](s)):
        y = host.group_norm_act(groups=2, act="none", eps=1e-3, p=0.25, rng=rng, **t)
    dy = torch.ones_like(y)
    host.launches.clear()
    for _ in range(2):
        torch.autograd.grad(y, x, dy, retain_graph=True)
        y.grad_fn.calls.clear()
    (_, one), (_, two) = host.launches
    assert bytes(one[0])[:-4] == bytes(two[0])[:-4] and one[1:3] == two[1:3] and one[-1] == two[-1]
    host.launches.clear()
    for bad in (lambda s: s.half() if s.is_floating_point() and s.dim() > 2 and s.shape[-1] > 2 else s,
                lambda s: torch.cat([s, s], 1) if s.dim() > 2 and s.shape[-1] > 2 else s, lambda s: s[:1] if s.shape[0] == n else s):
        y.grad_fn.calls.clear()
        swap[0] = bad
        with pytest.raises(ValueError):
            torch.autograd.grad(y, x, dy, retain_graph=True)
    assert not host.launches
