"""GPU tests of ivid_amd.functional against the 64-bit references and bounds of functional_ref.py."""
import numpy as np
import pytest
import torch

import common  # noqa: F401
import functional_ref as R

pytestmark = pytest.mark.gpu
DTS = [torch.float32, torch.bfloat16, torch.float16]
RNG = (0x123456789ABCDEF1, 7)


def F():
    from ivid_amd import functional
    return functional


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to("cuda", dtype)


def gn_inputs(seed, shape, c0, c1, dtype, film, offset=0.5):
    """x [*shape, c0], skip, weight, bias, film; shape[0] = N."""
    c = c0 + c1

    def act(s, ch):
        x = randn(s, *shape, ch) * (0.5 + torch.rand(ch, generator=torch.Generator().manual_seed(s + 1)).cuda()) + offset * randn(s + 2, ch)
        return x.to(dtype)
    return dict(x=act(seed, c0), skip=act(seed + 10, c1) if c1 else None, weight=1 + 0.2 * randn(seed + 20, c),
                bias=0.2 * randn(seed + 21, c),
                film=None if film is None else (0.3 * randn(seed + 22, shape[0], 2 * c)).to(dtype if film == "same" else torch.float32))


def run_gn(t, groups, dy, **kw):
    """(outputs as functional_ref names them) through autograd."""
    names = [k for k in ("x", "skip", "weight", "bias", "film") if t[k] is not None]
    leaves = {k: t[k].detach().requires_grad_() for k in names}
    y = F().group_norm_act(leaves["x"], groups, leaves["weight"], leaves["bias"], film=leaves.get("film"), skip=leaves.get("skip"), **kw)
    out = dict(y=y)
    out.update(zip(["d" + k for k in names], torch.autograd.grad(y, list(leaves.values()), dy)))
    with torch.no_grad():
        y2, out["stats"] = F().group_norm_act_forward(t["x"], groups, t["weight"], t["bias"], film=t["film"], skip=t["skip"], **kw)
    assert torch.equal(torch.nan_to_num(y2), torch.nan_to_num(y.detach()))
    return out


GN_CASES = [
    # name, [N, spatial...], C0, C1, groups, film, act, p
    ("one_value_a_group", (3, 1), 8, 0, 8, "f32", "silu", 0.0),
    ("two_values_a_group", (2, 1), 64, 0, 32, None, "silu", 0.0),
    ("one_pixel", (5, 1), 96, 0, 4, "same", "silu", 0.1),
    ("one_channel", (2, 9, 7), 1, 0, 1, "f32", "none", 0.3),
    ("bottleneck", (1, 8, 8), 1024, 0, 32, "f32", "silu", 0.0),
    ("plain_16x16", (3, 16, 16), 256, 0, 32, "same", "silu", 0.1),
    ("concat_seam_in_a_group", (2, 16, 16), 128, 96, 32, None, "silu", 0.0),
    ("concat_odd", (2, 5, 3), 33, 18, 17, "f32", "silu", 0.2),
    ("odd_37x23_c100_g20", (2, 37, 23), 100, 0, 20, "f32", "silu", 0.25),
    ("odd_c33_g3", (2, 13, 11), 33, 0, 3, "same", "silu", 0.1),
    ("c36_g6_seq77", (4, 77), 36, 0, 6, None, "none", 0.0),
    ("one_group_c513", (2, 6, 5), 513, 0, 1, "f32", "silu", 0.1),
    ("one_group_c1000", (1, 40, 12), 1000, 0, 1, None, "silu", 0.0),
    ("one_group_wide", (2, 3, 3), 5000, 0, 1, "f32", "silu", 0.5),
    ("one_channel_a_group", (2, 12, 12), 64, 0, 64, None, "silu", 0.0),
    ("one_channel_a_group_c200", (2, 9, 30), 200, 0, 200, "f32", "silu", 0.1),
    ("level0_64x64", (2, 64, 64), 64, 0, 32, "f32", "silu", 0.1),
    ("seq1024_c512", (2, 1024), 512, 0, 32, None, "none", 0.0),
    ("tall_128x128", (1, 128, 128), 128, 0, 32, "f32", "silu", 0.0),
    ("ragged_131x127_c48", (1, 131, 127), 48, 0, 8, None, "silu", 0.1),
    ("p_one", (2, 4, 4), 32, 0, 8, "f32", "silu", 1.0),
    ("many_samples", (300, 2, 2), 32, 0, 8, "f32", "silu", 0.1),
    ("tokens_2d", (5000,), 96, 0, 8, None, "silu", 0.1),
    ("tokens_odd_count", (1037, 1), 40, 24, 4, "same", "none", 0.0),
]


@pytest.mark.parametrize("dtype", DTS, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", GN_CASES, ids=[c[0] for c in GN_CASES])
def test_group_norm_act_and_its_gradients(case, dtype):
    name, shape, c0, c1, groups, film, act, p = case
    t = gn_inputs(sum(map(ord, name)), shape, c0, c1, dtype, film)
    dy = randn(5, *shape, c0 + c1, dtype=dtype)
    kw = dict(act=act, p=p, rng=RNG if p else None)
    want, bound = R.gn_act(t["x"], groups, t["weight"], t["bias"], film=t["film"], skip=t["skip"], dy=dy, **kw)
    got = run_gn(t, groups, dy, **kw)
    print(name, "worst ratio", R.check(got, want, bound, name))


def test_one_value_a_group_has_no_gradient():
    t = gn_inputs(3, (4, 1), 16, 0, torch.float32, "f32")
    got = run_gn(t, 16, randn(1, 4, 1, 16), act="silu")
    assert torch.equal(got["dx"], torch.zeros_like(got["dx"]))
    assert torch.equal(got["dweight"], torch.zeros_like(got["dweight"]))


@pytest.mark.parametrize("dtype", DTS, ids=["f32", "bf16", "f16"])
def test_large_mean_keeps_its_variance(dtype):
    """mean / deviation = 1000 (64 in the 16-bit types, whose steps would swallow the deviation): a sum of squares would lose it."""
    off = 1000.0 if dtype == torch.float32 else 64.0
    x = (randn(1, 2, 24, 24, 64) + off).to(dtype)
    t = dict(x=x, skip=None, weight=torch.ones(64, device="cuda"), bias=torch.zeros(64, device="cuda"), film=None)
    dy = randn(2, 2, 24, 24, 64, dtype=dtype)
    want, bound = R.gn_act(x, 8, t["weight"], t["bias"], dy=dy)
    R.check(run_gn(t, 8, dy), want, bound)


@pytest.mark.parametrize("dtype", DTS, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["channel_slice", "channel_slice_odd", "nchw", "channels_last", "misaligned", "row_slice", "expanded"])
def test_strided_inputs(layout, dtype):
    n, h, w, c, groups = 2, 10, 6, 48, 6
    if layout == "channel_slice":
        x = randn(1, n, h, w, 2 * c, dtype=dtype)[..., 16:16 + c]
    elif layout == "channel_slice_odd":
        x = randn(1, n, h, w, c + 5, dtype=dtype)[..., 3:3 + c]
    elif layout == "nchw":
        x = randn(1, n, c, h, w, dtype=dtype).permute(0, 2, 3, 1)
    elif layout == "channels_last":
        x = randn(1, n, c, h, w, dtype=dtype).to(memory_format=torch.channels_last).permute(0, 2, 3, 1)
    elif layout == "misaligned":
        x = randn(1, n * h * w * c + 1, dtype=dtype)[1:].view(n, h, w, c)
    elif layout == "row_slice":
        x = randn(1, n, h + 3, w + 2, c, dtype=dtype)[:, 1:h + 1, :w]
    else:
        x = randn(1, 1, h, w, c, dtype=dtype).expand(n, h, w, c)
    film = randn(3, n, 3 * 2 * c + 1)[:, c:3 * c] * 0.3
    t = dict(x=x, skip=None, weight=1 + randn(4, 2 * c)[::2] * 0.2, bias=randn(5, c) * 0.2, film=film)
    dy = randn(6, n, c, h, w, dtype=dtype).permute(0, 2, 3, 1)
    kw = dict(act="silu", p=0.2, rng=RNG)
    want, bound = R.gn_act(t["x"], groups, t["weight"], t["bias"], film=film, dy=dy, **kw)
    R.check(run_gn(t, groups, dy, **kw), want, bound, layout)


def test_strided_skip_and_source_give_what_the_concatenation_gives():
    base = randn(1, 2, 8, 8, 200, dtype=torch.bfloat16)
    x, skip = base[..., :72], base[..., 80:136]
    w, b = 1 + 0.1 * randn(2, 128), randn(3, 128)
    cat = torch.cat([x, skip], -1)
    a = F().group_norm_act(x, 16, w, b, skip=skip)
    assert torch.equal(a, F().group_norm_act(cat, 16, w, b))
    assert torch.equal(a, F().group_norm_act(x.contiguous(), 16, w, b, skip=skip.contiguous()))


def test_non_finite_values_stay_in_their_group():
    x = randn(1, 3, 6, 6, 32)
    x[1, 2, 3, 5] = float("nan")
    x[2, 0, 0, 31] = float("inf")
    w, b = torch.ones(32, device="cuda"), torch.zeros(32, device="cuda")
    dy = randn(2, 3, 6, 6, 32)
    t = dict(x=x, skip=None, weight=w, bias=b, film=None)
    got = run_gn(t, 4, dy)
    bad = torch.zeros(3, 4, dtype=torch.bool)
    bad[1, 0] = bad[2, 3] = True
    for k in ("y", "dx"):
        groups_bad = ~torch.isfinite(got[k].detach()).reshape(3, 36, 4, 8).all(3).all(1).cpu()
        assert torch.equal(groups_bad, bad), k


def test_extreme_activations_do_not_turn_into_nan():
    """v = +-200: the exponential overflows, silu is v or 0 and its slope 1 or 0."""
    x = randn(1, 2, 8, 8, 32)
    t = dict(x=x, skip=None, weight=torch.ones(32, device="cuda"), bias=torch.tensor([200.0, -200.0] * 16, device="cuda"), film=None)
    dy = randn(2, 2, 8, 8, 32)
    want, bound = R.gn_act(x, 4, t["weight"], t["bias"], dy=dy)
    R.check(run_gn(t, 4, dy), want, bound)


@pytest.mark.parametrize("p", [0.0, 0.3])
def test_gradients_against_differences(p):
    """The loss sum(y * r) in 64-bit sums of fp32 results: a central difference of step 2^-6 along a random direction is off by the
    rounding of y (bounded) / step plus step^2 / 6 times the third derivative; the direction is normalised, so both stay below
    1e-3 of the gradients' norm here."""
    n, h, w, c, g = 2, 6, 5, 32, 8
    t = gn_inputs(7, (n, h, w), c, 0, torch.float32, "f32")
    r = randn(9, n, h, w, c)
    kw = dict(p=p, rng=RNG if p else None)
    got = run_gn(t, g, r, **kw)
    for i, k in enumerate(("x", "weight", "bias", "film")):
        d = randn(20 + i, *t[k].shape)
        d /= d.norm()
        step = 2.0 ** -6
        val = []
        for s in (step, -step):
            q = dict(t, **{k: t[k] + s * d})
            y = F().group_norm_act(q["x"], g, q["weight"], q["bias"], film=q["film"], **kw)
            val.append((y.double() * r.double()).sum().item())
        fd = (val[0] - val[1]) / (2 * step)
        an = (got["d" + k].double() * d.double()).sum().item()
        assert abs(fd - an) <= 1e-3 * got["d" + k].double().norm().item(), (k, fd, an)


def test_only_the_gradients_asked_for():
    t = gn_inputs(8, (2, 4, 4), 32, 32, torch.float32, "f32")
    skip = t["skip"].requires_grad_()
    y = F().group_norm_act(t["x"], 8, t["weight"], t["bias"], film=t["film"], skip=skip)
    y.sum().backward()
    assert skip.grad.shape == skip.shape and t["x"].grad is None
    with pytest.raises(RuntimeError):      # differentiable once
        w = t["weight"].requires_grad_()
        (gw,) = torch.autograd.grad(F().group_norm_act(t["x"], 8, w, t["bias"], skip=skip).sum(), w, create_graph=True)
        gw.sum().backward()


def test_repeatable_and_independent_of_the_batch():
    t = gn_inputs(11, (24, 32, 32), 128, 0, torch.bfloat16, "f32")
    dy = randn(12, 24, 32, 32, 128, dtype=torch.bfloat16)
    a, b = run_gn(t, 32, dy), run_gn(t, 32, dy)
    for k in a:
        assert torch.equal(a[k], b[k]), k
    one = {k: (v[5:6] if k in ("x", "film") else v) for k, v in t.items()}
    c = run_gn(one, 32, dy[5:6])
    for k in ("y", "dx", "dfilm", "stats"):
        assert torch.equal(a[k][5:6], c[k]), k


@pytest.mark.parametrize("dtype", DTS, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 63, 4096, 100003])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(n, p, dtype):
    x = randn(n, n, dtype=dtype).requires_grad_()
    dy = randn(n + 1, n, dtype=dtype)
    y = F().dropout(x, p, RNG)
    (dx,) = torch.autograd.grad(y, x, dy)
    f = R.drop_factor(n, p, RNG)
    for got, src in ((y, x), (dx, dy)):
        want = src.detach().double().cpu() * f
        got = got.detach().double().cpu()
        assert torch.equal(got == 0, want == 0)
        # half a step of the type (below fp16's normal range steps are 2^-24 whatever the value), of the fp32 scale and product
        assert bool(((got - want).abs() <= want.abs() * (R.HALF[dtype] * 1.001 + 2 * R.U) + R.TINY[dtype]).all())


def test_dropout_draws_are_the_published_generator_at_far_indices():
    """Element 2^32 + k of a tensor longer than 2^32: 64-bit indices all the way (8.6 GB in, 8.6 GB out)."""
    n = (1 << 32) + 1027
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = F().dropout(x, 0.5, RNG)
    for first, count in ((0, 64), ((1 << 32) - 64, 1024 + 67)):
        want = R.draws(count, RNG, first) >= 32768
        assert np.array_equal((y[first:first + count] != 0).cpu().numpy(), want)
    del x, y
    torch.cuda.empty_cache()


def test_dropout_statistics_and_streams():
    n = 1 << 22
    x = torch.ones(n, device="cuda")
    a = F().dropout(x, 0.1, (1, 2))
    # kept ~ Binomial(n, 0.9): 6 deviations
    assert abs((a != 0).double().mean().item() - (1 - 6554 / 65536)) < 6 * (0.09 / n) ** 0.5
    assert abs(a.double().mean().item() - 1) < 6 * (0.09 / n) ** 0.5 / 0.9
    for other in ((1, 3), (2, 2), (1 + (1 << 40), 2), (1, 2 + (1 << 35))):
        b = F().dropout(x, 0.1, other)
        both = ((a != 0) == (b != 0)).double().mean().item()        # independent: 0.81 + 0.01
        assert abs(both - 0.82) < 6 * (0.82 * 0.18 / n) ** 0.5 + 1e-4
    assert torch.equal(a, F().dropout(x, 0.1, (1, 2)))


def test_dropout_layouts_and_non_finite_values():
    x = randn(1, 40, 30)
    f = R.drop_factor(1200, 0.3, RNG).reshape(40, 30)
    y = F().dropout(x.t(), 0.3, RNG).cpu()
    assert torch.equal(y == 0, R.drop_factor(1200, 0.3, RNG).reshape(30, 40) == 0)
    v = randn(2, 1201)[1:].view(40, 30)
    assert torch.equal(F().dropout(v, 0.3, RNG).cpu() == 0, f == 0)
    z = torch.full((40, 30), float("nan"), device="cuda")
    assert torch.equal(F().dropout(z, 0.3, RNG).cpu() == 0, f == 0)
    assert F().dropout(torch.empty(0, 5, device="cuda"), 0.5, RNG).shape == (0, 5)


def test_block_as_a_resblock_uses_it():
    """norm -> FiLM -> SiLU -> dropout in one call = the norm without dropout followed by `dropout` with the same rng (fp32: the
    scale multiplies the same fp32 value), forward and backward."""
    t = gn_inputs(31, (3, 9, 5), 40, 0, torch.float32, "f32")
    x = t["x"].requires_grad_()
    dy = randn(2, 3, 9, 5, 40)
    a = F().group_norm_act(x, 10, t["weight"], t["bias"], film=t["film"], p=0.2, rng=RNG)
    b = F().dropout(F().group_norm_act(x, 10, t["weight"], t["bias"], film=t["film"]), 0.2, RNG)
    assert torch.equal(a, b)
    ga, gb = torch.autograd.grad(a, x, dy)[0], torch.autograd.grad(b, x, dy)[0]
    assert torch.equal(ga, gb)


def test_empty_inputs():
    w, b = torch.ones(32, device="cuda").requires_grad_(), torch.zeros(32, device="cuda")
    for shape in ((0, 4, 4, 32), (2, 0, 4, 32)):
        x = torch.empty(shape, device="cuda").requires_grad_()
        y = F().group_norm_act(x, 8, w, b)
        assert y.shape == shape
        gx, gw = torch.autograd.grad(y, [x, w], torch.empty(shape, device="cuda"))
        assert gx.shape == shape and torch.equal(gw, torch.zeros_like(gw))


def test_on_another_stream():
    t = gn_inputs(41, (8, 32, 32), 256, 0, torch.bfloat16, "f32")
    dy = randn(3, 8, 32, 32, 256, dtype=torch.bfloat16)
    ref = run_gn(t, 32, dy, p=0.1, rng=RNG)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run_gn(t, 32, dy, p=0.1, rng=RNG)
    s.synchronize()
    for k in ref:
        assert torch.equal(ref[k], got[k]), k


def test_two_streams_at_once():
    ts = [gn_inputs(50 + i, (16, 64, 64), 128, 0, torch.bfloat16, "f32") for i in range(2)]
    dys = [randn(60 + i, 16, 64, 64, 128, dtype=torch.bfloat16) for i in range(2)]
    refs = [run_gn(t, 32, dy) for t, dy in zip(ts, dys)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run_gn(ts[i], 32, dys[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for k in refs[i]:
                assert torch.equal(refs[i][k], g[k]), (i, k)


def test_captured_step_replays_with_new_inputs_and_new_draws():
    """Forward and backward by hand in one graph, the draws from a device rng; every replay equals the eager result, with eager
    work of the same operators between the replays."""
    f = F()
    t = gn_inputs(71, (4, 64, 64), 64, 0, torch.bfloat16, "f32")
    dy = randn(72, 4, 64, 64, 64, dtype=torch.bfloat16)
    rng = torch.tensor([5, 6], device="cuda")
    args = (32, t["weight"], t["bias"])

    def step():
        y, stats = f.group_norm_act_forward(t["x"], *args, film=t["film"], p=0.1, rng=rng)
        z = f.dropout(y, 0.2, rng)
        dz = f.dropout(dy, 0.2, rng)
        return (y, z) + f.group_norm_act_backward(dz, stats, t["x"], *args, film=t["film"], p=0.1, rng=rng)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    seen = []
    for i in range(5):
        t["x"].copy_(randn(80 + i, 4, 64, 64, 64))
        rng.copy_(torch.tensor([5 + i, 6]))
        graph.replay()
        got = [o.clone() for o in out if o is not None]
        want = [o for o in step() if o is not None]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        seen.append(got[1] == 0)
    assert not torch.equal(seen[0], seen[1])


def test_two_graphs_replayed_at_once():
    f = F()
    ts = [gn_inputs(90 + i, (8, 64, 64), 128, 0, torch.bfloat16, "f32") for i in range(2)]
    dys = [randn(95 + i, 8, 64, 64, 128, dtype=torch.bfloat16) for i in range(2)]
    graphs, outs, wants = [], [], []
    for t, dy in zip(ts, dys):
        def step(t=t, dy=dy):
            y, stats = f.group_norm_act_forward(t["x"], 32, t["weight"], t["bias"], film=t["film"])
            return (y,) + f.group_norm_act_backward(dy, stats, t["x"], 32, t["weight"], t["bias"], film=t["film"])
        wants.append([o.clone() for o in step() if o is not None])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, wants):
            for a, b in zip([q for q in o if q is not None], w):
                assert torch.equal(a, b)


def test_autograd_through_leaves_is_refused_under_capture():
    from ivid_amd._lib import IvidHipError
    x = randn(1, 2, 4, 4, 32).requires_grad_()
    w, b = torch.ones(32, device="cuda"), torch.zeros(32, device="cuda")
    g = torch.cuda.CUDAGraph()
    refused = []
    with torch.cuda.graph(g):
        for fn in (lambda: F().group_norm_act(x, 8, w, b), lambda: F().dropout(x, 0.5, RNG)):
            try:
                fn()
            except IvidHipError as e:
                refused.append(str(e))
        keep = w + 1  # noqa: F841  (a graph with a node)
    assert len(refused) == 2
    assert F().group_norm_act(x, 8, w, b).requires_grad


def test_autograd_behind_a_leaf_is_refused_under_capture():
    from ivid_amd._lib import IvidHipError
    leaf = randn(1, 2, 4, 4, 32).requires_grad_()
    x = leaf * 2
    w, b = torch.ones(32, device="cuda"), torch.zeros(32, device="cuda")
    g = torch.cuda.CUDAGraph()
    refused = 0
    with torch.cuda.graph(g):
        for fn in (lambda: F().group_norm_act(x, 8, w, b), lambda: F().dropout(x, 0.5, RNG)):
            try:
                fn()
            except IvidHipError:
                refused += 1
        with torch.no_grad():
            y = F().dropout(F().group_norm_act(x, 8, w, b), 0.5, RNG)
    assert refused == 2
    g.replay()
    assert torch.equal(y, F().dropout(F().group_norm_act(x, 8, w, b), 0.5, RNG))


def test_a_rewritten_rng_tensor_is_noticed():
    x = randn(1, 100).requires_grad_()
    rng = torch.tensor([1, 2], device="cuda")
    y = F().dropout(x, 0.5, rng)
    rng.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("dtype", DTS, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,c0,c1,groups", [((3, 7, 5), 24, 0, 6), ((2, 33), 50, 14, 8), ((2, 40, 41), 64, 0, 32), ((1, 70, 70), 72, 0, 9)])
def test_nothing_is_written_outside_the_outputs(shape, c0, c1, groups, dtype):
    """Every output and the scratch sit between guard bytes."""
    import ctypes
    from ivid_amd import _lib
    f = F()
    t = gn_inputs(101, shape, c0, c1, dtype, "same")
    c = c0 + c1
    call = f._Call(t["x"], groups, t["weight"], t["bias"], t["film"], t["skip"], "silu", 1e-5, 0.1, RNG)
    pix = t["x"].numel() // c0
    esz = t["x"].element_size()
    guarded = []

    def buf(nbytes):
        b = torch.full((nbytes + 512,), 0xA5, dtype=torch.uint8, device="cuda")
        guarded.append((b, nbytes))
        return b.data_ptr() + 256
    lib = _lib.load()
    st = torch.cuda.current_stream().cuda_stream
    nb = [lib.ivid_gn_act_scratch_bytes(ctypes.byref(call.desc), i) for i in range(2)]
    stats = buf(shape[0] * groups * 8)
    _lib.call("ivid_gn_act_forward", ctypes.byref(call.desc), buf(pix * c * esz), stats, buf(nb[0]), nb[0], st)
    dy = randn(7, *shape, c, dtype=dtype)
    _lib.call("ivid_gn_act_backward", ctypes.byref(call.desc), stats, dy.data_ptr(), buf(pix * c0 * esz), buf(pix * c1 * esz) if c1 else None,
              buf(4 * c), buf(4 * c), buf(shape[0] * 2 * c * esz), buf(nb[1]), nb[1], st)
    n = pix * c + 3
    x = randn(8, n, dtype=dtype)
    _lib.call("ivid_dropout", f._DTYPES[dtype], x.data_ptr(), buf(n * esz), n, 0.5, 1, 2, None, st)
    torch.cuda.synchronize()
    for b, nbytes in guarded:
        assert bool((b[:256] == 0xA5).all()) and bool((b[256 + nbytes:] == 0xA5).all())


@pytest.mark.parametrize("dtype", DTS, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,c0,c1,groups", [((3, 64, 64), 128, 0, 32), ((2, 61, 67), 50, 0, 10), ((2, 50, 50), 1000, 24, 1), ((1, 128, 128), 33, 0, 3)])
def test_a_workgroup_that_stops_waiting_changes_nothing(shape, c0, c1, groups, dtype, monkeypatch):
    """One poll: workgroups compute the sums that have not come yet themselves; every output is the same bit for bit."""
    t = gn_inputs(111, shape, c0, c1, dtype, "f32")
    dy = randn(112, *shape, c0 + c1, dtype=dtype)
    ref = run_gn(t, groups, dy, p=0.1, rng=RNG)
    monkeypatch.setattr(F(), "_MAX_POLLS", 1)
    for _ in range(3):
        got = run_gn(t, groups, dy, p=0.1, rng=RNG)
        for k in ref:
            assert torch.equal(ref[k], got[k]), k
    want, bound = R.gn_act(t["x"], groups, t["weight"], t["bias"], film=t["film"], skip=t["skip"], dy=dy, p=0.1, rng=RNG)
    R.check(ref, want, bound)


def test_offsets_beyond_32_bits():
    """6.4e9 values in one call (12.9 GB a tensor): the last sample equals the call on it alone."""
    n, hw, c = 3, 1 << 24, 128
    x = torch.empty(n, hw, c, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    w, b = 1 + 0.1 * randn(2, c), randn(3, c)
    y, stats = F().group_norm_act_forward(x, 32, w, b)
    y1, stats1 = F().group_norm_act_forward(x[2:], 32, w, b)
    assert torch.equal(y[2:], y1) and torch.equal(stats[2:], stats1)
    assert abs(stats[..., 0].abs().max().item()) < 1e-3 and (stats[..., 1] - 1).abs().max().item() < 1e-3
    del y1
    dx = F().group_norm_act_backward(x, stats, x, 32, w, b)[0]
    dx1 = F().group_norm_act_backward(x[2:], stats1, x[2:], 32, w, b)[0]
    assert torch.equal(dx[2:], dx1)
    del x, y, dx, dx1
    torch.cuda.empty_cache()


def test_backward_twice_and_one_tensor_in_two_places():
    t = gn_inputs(121, (2, 9, 9), 48, 0, torch.float32, "f32")
    x, w = t["x"].requires_grad_(), (1 + 0.1 * randn(1, 96)).requires_grad_()
    b = randn(2, 96) * 0.1
    film = (0.3 * randn(3, 1, 192)).requires_grad_()
    dy = randn(4, 2, 9, 9, 96)
    rng = torch.tensor([3, 4], device="cuda")
    y = F().group_norm_act(x, 12, w, b, film=film.expand(2, 192), skip=x, p=0.1, rng=rng)
    a = torch.autograd.grad(y, [x, w, film], dy, retain_graph=True)
    c = torch.autograd.grad(y, [x, w, film], dy)
    for p, q in zip(a, c):
        assert torch.equal(p, q)
    want, bound = R.gn_act(x, 12, w, b, film=film.expand(2, 192), skip=x, dy=dy, p=0.1, rng=(3, 4))
    got = dict(y=y, dx=a[0], dweight=a[1], dfilm=a[2])
    for k, both in (("dx", "dskip"), ("dfilm", None)):
        if both:
            want[k], bound[k] = want[k] + want[both], bound[k] + bound[both] + R.U * (want[k].abs() + want[both].abs())
        else:
            want[k], bound[k] = want[k].sum(0, keepdim=True), bound[k].sum(0, keepdim=True) + 2 * R.U * want[k].abs().sum(0, keepdim=True)
    R.check(got, {k: want[k] for k in got}, bound)


def test_saved_tensors_may_be_moved_or_recomputed():
    from torch.utils.checkpoint import checkpoint
    t = gn_inputs(131, (3, 20, 20), 64, 0, torch.bfloat16, "f32")
    x, w, b, film = t["x"].requires_grad_(), t["weight"].requires_grad_(), t["bias"].requires_grad_(), t["film"].requires_grad_()
    dy = randn(5, 3, 20, 20, 64, dtype=torch.bfloat16)

    def block(x, w, b, film):
        return F().dropout(F().group_norm_act(x, 8, w, b, film=film, p=0.1, rng=RNG), 0.2, (9, 9))
    ref = torch.autograd.grad(block(x, w, b, film), [x, w, b, film], dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s.cpu(), lambda s: s.cuda()):
        y = block(x, w, b, film)
    for p, q in zip(ref, torch.autograd.grad(y, [x, w, b, film], dy)):
        assert torch.equal(p, q)
    y = checkpoint(block, x, w, b, film, use_reentrant=False)
    for p, q in zip(ref, torch.autograd.grad(y, [x, w, b, film], dy)):
        assert torch.equal(p, q)


@pytest.mark.parametrize("layout", ["offset", "pixel stride", "both strides"])
def test_saved_tensors_may_come_back_with_other_strides_and_alignment(layout):
    """The backward pass is cut by the strides and the alignment of the tensors that it gets, not by those of the forward call."""
    n, hw, c = 2, 1300, 64
    if layout == "offset":
        x = randn(3, n * hw * c + 1, dtype=torch.bfloat16)[1:].view(n, hw, c)
    elif layout == "pixel stride":
        x = randn(3, n, hw, c + 1, dtype=torch.bfloat16)[..., :c]
    else:
        x = randn(3, n, hw + 1, c + 3, dtype=torch.bfloat16)[:, 1:, 3:]
    x, w, b, dy = x.detach().requires_grad_(), randn(4, c).requires_grad_(), randn(5, c).requires_grad_(), randn(6, n, hw, c, dtype=torch.bfloat16)
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s, lambda s: s.clone(memory_format=torch.contiguous_format)):
        y = F().group_norm_act(x, 8, w, b, p=0.1, rng=RNG)
    want, bound = R.gn_act(x.detach(), 8, w.detach(), b.detach(), p=0.1, rng=RNG, dy=dy)
    got = dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, [x, w, b], dy)))
    R.check(got, {k: want[k] for k in got}, bound)


def test_a_constant_sample():
    """No variance: xhat is 0 to the rounding of the mean, rstd 1 / sqrt(eps) -- 10^4 with eps = 10^-8 --, and nothing is NaN."""
    x = torch.full((2, 17, 64), 3.0, device="cuda")
    x[1] = 0
    w, b = torch.ones(64, device="cuda"), randn(1, 64)
    for eps in (1e-5, 1e-8):
        want, bound = R.gn_act(x, 8, w, b, eps=eps)
        y, stats = F().group_norm_act_forward(x, 8, w, b, eps=eps)
        R.check(dict(y=y, stats=stats), want, bound)
        assert torch.isfinite(y).all()
    dx = F().group_norm_act_backward(randn(2, 2, 17, 64), stats, x, 8, w, b, eps=1e-8)[0]
    assert torch.isfinite(dx).all()


def test_python_entry_points_refuse_what_does_not_fit():
    f = F()
    x, w, b = randn(1, 2, 4, 32), torch.ones(32, device="cuda"), torch.zeros(32, device="cuda")
    bad = [(ValueError, dict(groups=5)), (ValueError, dict(groups=0)), (TypeError, dict(weight=w.half())), (ValueError, dict(weight=w[:16])),
           (ValueError, dict(bias=b.cpu())), (ValueError, dict(film=randn(1, 2, 32))), (TypeError, dict(film=randn(1, 2, 64).double())),
           (ValueError, dict(film=randn(1, 3, 64))), (ValueError, dict(skip=randn(1, 2, 5, 32))), (ValueError, dict(skip=randn(1, 2, 4, 8).half())),
           (ValueError, dict(skip=randn(1, 2, 4, 0))), (ValueError, dict(act="gelu")), (ValueError, dict(eps=0.0)),
           (ValueError, dict(eps=float("inf"))), (ValueError, dict(p=1.5, rng=RNG)), (ValueError, dict(p=0.5)),
           (ValueError, dict(p=0.5, rng=torch.zeros(2, dtype=torch.int32, device="cuda"))),
           (ValueError, dict(p=0.5, rng=torch.zeros(2, dtype=torch.int64))), (TypeError, dict(x=x.double())), (ValueError, dict(x=randn(1, 32)))]
    for err, kw in bad:
        args = dict(dict(x=x, groups=8, weight=w, bias=b), **kw)
        with pytest.raises(err):
            f.group_norm_act(**args)
    one = torch.ones(1, device="cuda")
    for huge in (one.expand(1, (1 << 32) + 4, 1), one.expand((1 << 32) + 4, 1, 1)):      # sizes that would wrap to 4
        with pytest.raises(ValueError):
            f.group_norm_act(huge, 1, one, one)
    y, stats = f.group_norm_act_forward(x, 8, w, b)
    for dy, st in ((y[:1], stats), (y.half(), stats), (y, stats[:1]), (y, stats.double()), (y.cpu(), stats)):
        with pytest.raises(ValueError):
            f.group_norm_act_backward(dy, st, x, 8, w, b)
    dy = torch.empty(2 * 4 * 32 + 1, device="cuda")[1:].view(2, 4, 32).copy_(y)      # a gradient that is not on 16 bytes
    for p, q in zip(f.group_norm_act_backward(dy, stats, x, 8, w, b), f.group_norm_act_backward(y, stats, x, 8, w, b)):
        assert (p is None and q is None) or torch.equal(p, q)


def test_dropout_without_draws_has_a_gradient():
    """p = 0 needs no rng, in the backward pass either; an empty tensor has nothing to draw."""
    for shape, p in (((40, 30), 0.0), ((0, 5), 0.0), ((0, 5), 0.5)):
        x = torch.empty(shape, device="cuda").normal_().requires_grad_()
        dy = torch.empty(shape, device="cuda").normal_()
        y = F().dropout(x, p)
        (dx,) = torch.autograd.grad(y, x, dy)
        assert torch.equal(y, x) and torch.equal(dx, dy)


def test_saved_tensors_that_come_back_elsewhere_are_refused():
    t = gn_inputs(141, (2, 6, 6), 32, 32, torch.bfloat16, "f32")
    x = t["x"].requires_grad_()
    for name in ("x", "skip", "weight", "bias", "film", "stats"):
        shape = t[name].shape if name in t else (2, 8, 2)
        seen = []

        def unpack(s, shape=shape, name=name, seen=seen):
            if s.shape == shape and (name != "bias" or seen):      # (weight and bias have one shape; the weight comes first)
                return s.cpu()
            seen.extend([1] * (s.dim() == 1))
            return s
        with torch.autograd.graph.saved_tensors_hooks(lambda s: s, unpack):
            y = F().group_norm_act(x, 8, t["weight"], t["bias"], film=t["film"], skip=t["skip"])
        with pytest.raises(ValueError):
            torch.autograd.grad(y, x, torch.ones_like(y))


@pytest.mark.parametrize("dtype", DTS, ids=["f32", "bf16", "f16"])
def test_saved_tensors_may_come_back_transposed_in_memory(dtype):
    """Every saved tensor, the statistics among them, with its first and last dimension swapped in memory."""
    t = gn_inputs(151, (3, 9, 7), 24, 16, dtype, "f32")
    dy = randn(152, 3, 9, 7, 40, dtype=dtype)
    names = ("x", "skip", "weight", "bias", "film")
    leaves = {k: t[k].requires_grad_() for k in names}
    kw = dict(p=0.2, rng=RNG)
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s, lambda s: s.transpose(0, -1).contiguous().transpose(0, -1)):
        y = F().group_norm_act(x=leaves["x"], groups=8, weight=leaves["weight"], bias=leaves["bias"], film=leaves["film"],
                               skip=leaves["skip"], **kw)
    got = dict(zip(["d" + k for k in names], torch.autograd.grad(y, list(leaves.values()), dy)), y=y)
    want, bound = R.gn_act(t["x"], 8, t["weight"], t["bias"], film=t["film"], skip=t["skip"], dy=dy, **kw)
    R.check(got, {k: want[k] for k in got}, bound)


def test_more_samples_than_one_launch_holds():
    """2^23 + 13 samples of a tile each: the forward pass takes two launches, and every sample is what it is in a call of fewer."""
    n, c = (1 << 23) + 13, 8
    x = torch.empty(n, c, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    w, b = 1 + 0.2 * randn(2, c), 0.2 * randn(3, c)
    y, stats = F().group_norm_act_forward(x, 1, w, b, p=0.25, rng=RNG)
    half = 1 << 22
    for i in range(0, n, half):
        y1, stats1 = F().group_norm_act_forward(x[i:i + half], 1, w, b)
        kept = y[i:i + half] != 0
        assert torch.equal(stats[i:i + half], stats1)
        assert abs(kept.float().mean().item() - 0.75) < 0.01
    for i in (0, half, (1 << 23) - 40, n - 64):
        count = min(64, n - i)
        want, bound = R.gn_act(x[i:i + count], 1, w, b)
        f = torch.from_numpy((R.draws(count * c, RNG, i * c) >= R.threshold(0.25)) * (4 / 3)).reshape(count, c)
        bound["y"], want["y"] = bound["y"] * f + 2 * R.U * (want["y"] * f).abs(), want["y"] * f
        R.check(dict(y=y[i:i + count], stats=stats[i:i + count]), want, bound)
    dy = torch.ones_like(x)
    dx = F().group_norm_act_backward(dy, stats, x, 1, w, b, p=0.25, rng=RNG)[0]
    del y, dy
    assert torch.isfinite(dx[::4099]).all()


def test_parameter_gradients_over_many_tiles():
    """One sample of 2^26 pixels, 16384 tiles that are all alike: their sums are equal terms, whose additions all round the same way.
    Every sum is 16384 times that over one tile, so is every bound."""
    tile, count = 4096, 1 << 14
    x = randn(1, 1, tile, 1, dtype=torch.bfloat16)
    dy = (1 + 0.5 * x.float() + 0.25 * randn(2, 1, tile, 1)).to(torch.bfloat16)
    w, b, film = 1 + 0.2 * randn(3, 1), 0.2 * randn(4, 1), 0.3 * randn(5, 1, 2)
    want, bound = R.gn_act(x, 1, w, b, film=film, dy=dy)
    whole = lambda t: t.expand(count, tile, 1).reshape(1, count * tile, 1)
    y, stats = F().group_norm_act_forward(whole(x), 1, w, b, film=film)
    dx, _, dw, db, dfilm = F().group_norm_act_backward(whole(dy), stats, whole(x), 1, w, b, film=film)
    for i in (0, tile * 5461, tile * (count - 1)):
        R.check(dict(y=y[:, i:i + tile], dx=dx[:, i:i + tile], stats=stats), {k: want[k] for k in ("y", "dx", "stats")}, bound)
    got = dict(dweight=dw, dbias=db, dfilm=dfilm)
    print("worst ratio", R.check(got, {k: want[k] * count for k in got}, {k: bound[k] * count for k in got}))


def test_parameter_gradients_over_many_samples():
    """2^22 samples that are all alike, one pixel each; the same argument."""
    n, c = 1 << 22, 8
    x, dy = randn(1, 1, c), torch.tensor([[1.1, 0.7, 1.9, 0.3, 1.3, 1.23, 0.9, 1.7]], device="cuda")
    w, b = 1 + 0.2 * randn(3, c), 0.2 * randn(4, c)
    want, bound = R.gn_act(x, 1, w, b, dy=dy, act="none")
    y, stats = F().group_norm_act_forward(x.expand(n, c), 1, w, b, act="none")
    dx, _, dw, db, _ = F().group_norm_act_backward(dy.expand(n, c), stats, x.expand(n, c), 1, w, b, act="none")
    for t in (y, dx, stats):
        assert torch.equal(t, t[:1].expand_as(t))
    R.check(dict(y=y[:1], dx=dx[:1], stats=stats[:1]), {k: want[k] for k in ("y", "dx", "stats")}, bound)
    got = dict(dweight=dw, dbias=db)
    print("worst ratio", R.check(got, {k: want[k] * n for k in got}, {k: bound[k] * n for k in got}))


@pytest.mark.parametrize("dtype", DTS, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,c0,c1,groups,film,p", [((2, 1100003), 1, 1, 2, "f32", 0.1), ((1, 2200003), 1, 0, 1, None, 0.0)], ids=["skip", "one_channel"])
def test_more_tiles_than_one_launch_exchanges(shape, c0, c1, groups, film, p, dtype):
    """A sample of more than 256 tiles takes two launches, sums and results, in both directions."""
    t = gn_inputs(161, shape, c0, c1, dtype, film, offset=2.0)
    dy = 0.5 + randn(162, *shape, c0 + c1)
    dy = dy.to(dtype)
    kw = dict(act="silu", p=p, rng=RNG if p else None)
    want, bound = R.gn_act(t["x"], groups, t["weight"], t["bias"], film=t["film"], skip=t["skip"], dy=dy, **kw)
    got = run_gn(t, groups, dy, **kw)
    print("worst ratio", R.check(got, want, bound))


def test_more_tiles_than_one_launch_exchanges_in_several_slabs():
    t = gn_inputs(171, (1, 270001), 64, 0, torch.float32, None)
    dy = 0.5 + randn(172, 1, 270001, 64)
    want, bound = R.gn_act(t["x"], 32, t["weight"], t["bias"], dy=dy)
    print("worst ratio", R.check(run_gn(t, 32, dy), want, bound))


@pytest.mark.parametrize("dtype", DTS, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,c0,c1,film", [((40, 200), 5000, 0, "f32"), ((24, 150), 1000, 3096, "same")], ids=["c5000", "skip"])
def test_a_workgroup_that_stops_waiting_in_a_group_of_several_column_chunks(shape, c0, c1, film, dtype, monkeypatch):
    """One poll, and more workgroups than the chip holds: a workgroup adds up tiles of other channels than its own and has to come
    back to its own coefficients."""
    t = gn_inputs(181, shape, c0, c1, dtype, film)
    dy = randn(182, *shape, c0 + c1, dtype=dtype)
    ref = run_gn(t, 1, dy, p=0.1, rng=RNG)
    monkeypatch.setattr(F(), "_MAX_POLLS", 1)
    for _ in range(3):
        got = run_gn(t, 1, dy, p=0.1, rng=RNG)
        for k in ref:
            assert torch.equal(ref[k], got[k]), k
    one = {k: v[:1] if v is not None and k in ("x", "skip", "film") else v for k, v in t.items()}
    want, bound = R.gn_act(one["x"], 1, t["weight"], t["bias"], film=one["film"], skip=one["skip"], dy=dy[:1], p=0.1, rng=RNG)
    R.check({k: v[:1] for k, v in ref.items() if k not in ("dweight", "dbias")}, {k: v for k, v in want.items() if k not in ("dweight", "dbias")}, bound)


@pytest.mark.parametrize("dtype", DTS, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,c0,c1,groups", [((9, 37, 23), 100, 0, 20), ((7, 77), 36, 0, 6), ((5, 13, 11), 33, 0, 3), ((5, 40, 41), 18, 30, 6),
                                                ((3, 90, 91), 64, 0, 32), ((300, 1), 24, 0, 3)])
def test_independent_of_the_batch_at_odd_sizes(shape, c0, c1, groups, dtype):
    """A sample alone, as a view of the batch or as a copy, gives the bits that it gives among others."""
    t = gn_inputs(191, shape, c0, c1, dtype, "f32")
    dy = randn(192, *shape, c0 + c1, dtype=dtype)
    whole = run_gn(t, groups, dy)
    for i in (0, 1, shape[0] - 1):
        for copy in (False, True):
            pick = lambda v: v[i:i + 1].clone() if copy else v[i:i + 1]
            one = {k: pick(v) if v is not None and k in ("x", "skip", "film") else v for k, v in t.items()}
            got = run_gn(one, groups, pick(dy))
            for k in whole:
                if k not in ("dweight", "dbias"):
                    assert torch.equal(whole[k][i:i + 1], got[k]), (k, i, copy)


def test_dropout_probabilities_next_to_the_ends():
    """p is used in steps of 2^-16, rounded to the nearest: less than half a step drops nothing, less than half a step below 1 all."""
    x = randn(1, 1000)
    assert torch.equal(F().dropout(x, 2.0 ** -17 * 0.99, RNG), x)
    assert torch.equal(F().dropout(x, 1 - 2.0 ** -17, RNG), torch.zeros_like(x))
    keep = R.drop_factor(1 << 20, 1 - 2.0 ** -16, RNG)
    y = F().dropout(torch.ones(1 << 20, device="cuda"), 1 - 2.0 ** -16, RNG).double().cpu()
    assert torch.equal(y, keep) and 0 < int((y != 0).sum()) < 100
