"""CPU: what ivid_amd.functional and its C entry points refuse, and the references they are tested against."""
import ctypes

import numpy as np
import pytest
import torch

import functional_ref as R


def test_cpu_tensors_are_refused():
    from ivid_amd import functional as F
    from ivid_amd._lib import IvidHipError
    with pytest.raises(IvidHipError):
        F.dropout(torch.zeros(4), 0.5, (1, 2))
    with pytest.raises(IvidHipError):
        F.group_norm_act(torch.zeros(1, 4, 8), 2, torch.ones(8), torch.zeros(8))


def test_bad_types_and_probabilities_are_refused():
    from ivid_amd import functional as F
    with pytest.raises(TypeError):
        F.dropout(torch.zeros(4, dtype=torch.float64), 0.5, (1, 2))
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            F._check_p(p)
    dev = torch.device("cpu")
    for rng in (None, (-1, 0), (0, 1 << 64), torch.zeros(2), torch.zeros(3, dtype=torch.int64), torch.zeros(4, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError):
            F._rng_args(rng, 0.5, dev)
    assert F._rng_args(None, 0.0, dev) == (0, 0, None)


def _desc(**kw):
    from ivid_amd import _lib
    buf = np.zeros(64, np.float64).ctypes.data       # never dereferenced: every call here is refused on the host
    d = dict(dtype=_lib.F32, N=1, HW=4, C0=8, C1=0, groups=2, act=1, src0=buf, ld0=8, sn0=32, src1=None, ld1=0, sn1=0, gamma=buf,
             beta=buf, film=None, film_dtype=0, film_ld=0, eps=1e-5, p=0.0, seed=0, stream_id=0, rng=None)
    d.update(kw)
    return _lib.GnActDesc(**d), buf


BAD = [dict(dtype=3), dict(dtype=9), dict(N=-1), dict(HW=-1), dict(C0=0), dict(C1=-8), dict(groups=3), dict(groups=0), dict(groups=-2),
       dict(act=2), dict(eps=0.0), dict(eps=float("nan")), dict(p=-0.5), dict(p=1.01), dict(p=float("nan")), dict(C1=8), dict(src0=None),
       dict(gamma=None), dict(beta=None), dict(src0=4097), dict(gamma=4098), dict(rng=4100), dict(film=4096, film_dtype=2),
       dict(film=4097, film_dtype=0)]


@pytest.mark.parametrize("kw", BAD, ids=[str(k) for k in BAD])
def test_malformed_descriptors_are_refused(kw):
    from ivid_amd import _lib
    lib = _lib.load()
    d, buf = _desc(**kw)
    assert lib.ivid_gn_act_scratch_bytes(ctypes.byref(d), 0) == -1
    assert lib.ivid_gn_act_scratch_bytes(ctypes.byref(d), 1) == -1
    assert lib.ivid_gn_act_forward(ctypes.byref(d), buf, buf, buf, 1 << 20, None) != 0
    assert lib.ivid_last_error()
    assert lib.ivid_gn_act_backward(ctypes.byref(d), buf, buf, buf, None, buf, buf, None, buf, 1 << 20, None) != 0


def test_missing_outputs_and_short_scratch_are_refused():
    from ivid_amd import _lib
    lib = _lib.load()
    d, buf = _desc()
    fwd = lambda *a: lib.ivid_gn_act_forward(ctypes.byref(d), *a, None)
    bwd = lambda *a: lib.ivid_gn_act_backward(ctypes.byref(d), *a, None)
    assert lib.ivid_gn_act_forward(None, buf, buf, buf, 1 << 20, None) != 0
    assert fwd(None, buf, buf, 1 << 20) != 0
    assert fwd(buf, None, buf, 1 << 20) != 0
    need = lib.ivid_gn_act_scratch_bytes(ctypes.byref(d), 1)
    assert need > 0
    ok = [buf, buf, buf, None, buf, buf, None, buf, need]
    for i in (0, 1, 2, 4, 5, 7):
        bad = list(ok)
        bad[i] = None
        assert bwd(*bad) != 0, i
    assert bwd(*ok[:8], need - 1) != 0
    assert bwd(*ok[:3], buf, *ok[4:]) != 0           # dsrc1 without src1
    assert bwd(*ok[:6], buf, *ok[7:]) != 0           # dfilm without film


def test_dropout_entry_point_refuses_bad_arguments():
    from ivid_amd import _lib
    lib = _lib.load()
    buf = 1 << 20
    for args in ((3, buf, buf, 8, 0.5), (7, buf, buf, 8, 0.5), (0, buf, buf, -1, 0.5), (0, None, buf, 8, 0.5), (0, buf, None, 8, 0.5),
                 (0, buf + 2, buf, 8, 0.5), (1, buf, buf + 1, 8, 0.5), (0, buf, buf, 8, -0.1), (0, buf, buf, 8, 1.1),
                 (0, buf, buf, 8, float("nan"))):
        assert lib.ivid_dropout(*args, 1, 2, None, None) != 0, args
    assert lib.ivid_dropout(0, buf, buf, 8, 0.5, 1, 2, buf + 4, None) != 0
    assert lib.ivid_dropout(0, None, None, 0, 0.5, 1, 2, None, None) == 0


def test_eps_that_fp32_does_not_hold_is_refused():
    from ivid_amd import _lib
    lib = _lib.load()
    for eps in (1e-50, 1e39, float("inf"), -1e-5):
        d, _ = _desc(eps=eps)
        assert lib.ivid_gn_act_scratch_bytes(ctypes.byref(d), 0) == -1, eps


def _address(k):
    """16-byte aligned addresses that are never read: every call here is refused on the host"""
    return (1 << 24) + k


def test_overlapping_tensors_are_refused():
    from ivid_amd import _lib
    lib = _lib.load()
    msg = lambda: lib.ivid_last_error().decode()
    # one sample of 4 pixels x 8 channels fp32 (128 bytes), a second source of 8 channels behind it with pixels 16 floats apart
    ptr = dict(gamma=_address(1 << 16), beta=_address(1 << 16))
    d, _ = _desc(src0=_address(0), **ptr)
    for out in (0, 16, 112, -112):
        assert lib.ivid_gn_act_forward(ctypes.byref(d), _address(out), _address(1 << 17), None, 0, None) != 0
        assert "overlaps" in msg(), out
    for dx in (0, 4096, 4096 + 112):      # x, dy, the end of dy
        assert lib.ivid_gn_act_backward(ctypes.byref(d), _address(1 << 17), _address(4096), _address(dx), None, _address(1 << 18),
                                        _address(1 << 18), None, _address(1 << 19), 1 << 16, None) != 0
        assert "overlaps" in msg(), dx
    d, _ = _desc(src0=_address(0), C1=8, src1=_address(1024), ld1=16, sn1=64, **ptr)
    for out in (1024 + 3 * 64 + 16, 1024 - 240):       # the last pixel of the second source, its first from below
        assert lib.ivid_gn_act_forward(ctypes.byref(d), _address(out), _address(1 << 17), None, 0, None) != 0
        assert "overlaps" in msg(), out
    for d0, d1 in ((8192, 8192 + 112), (8192, 1024), (1024 + 16, 8192), (8192, 4096 + 240)):
        assert lib.ivid_gn_act_backward(ctypes.byref(d), _address(1 << 17), _address(4096), _address(d0), _address(d1), _address(1 << 18),
                                        _address(1 << 18), None, _address(1 << 19), 1 << 16, None) != 0
        assert "overlaps" in msg(), (d0, d1)
    for x, out in ((0, 16), (16, 0), (0, 28), (28, 0)):
        assert lib.ivid_dropout(0, _address(x), _address(out), 8, 0.5, 1, 2, None, None) != 0
        assert "overlap" in msg()


def test_reference_gradients_are_autograds():
    """The closed-form gradients of functional_ref against automatic differentiation in 64 bits."""
    g = torch.Generator().manual_seed(0)
    n, hw, c0, c1, groups, rng, p = 2, 6, 8, 4, 3, (3, 4), 0.3
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, skip, w, b, film, dy = mk(n, hw, c0), mk(n, hw, c1), mk(c0 + c1), mk(c0 + c1), mk(n, 2 * (c0 + c1)), mk(n, hw, c0 + c1)
    for t in (x, skip, w, b, film):
        t.requires_grad_()
    z = torch.cat([x, skip], -1).reshape(n, hw, groups, -1)
    z = (z - z.mean((1, 3), keepdim=True)) / (z.var((1, 3), unbiased=False, keepdim=True) + 1e-5).sqrt()
    v = (z.reshape(n, hw, -1) * w + b) * (1 + film[:, None, :c0 + c1]) + film[:, None, c0 + c1:]
    y = v * torch.sigmoid(v) * R.drop_factor(dy.numel(), p, rng).reshape(dy.shape)
    grads = torch.autograd.grad(y, [x, skip, w, b, film], dy)
    R_types = {torch.float64: 2.0 ** -53}
    R.HALF.update(R_types), R.TINY.update(R_types)
    try:
        out, _ = R.gn_act(x, groups, w, b, film=film, skip=skip, p=p, rng=rng, dy=dy)
    finally:
        R.HALF.pop(torch.float64), R.TINY.pop(torch.float64)
    assert torch.allclose(out["y"], y.detach(), atol=1e-12)
    for k, gr in zip(("dx", "dskip", "dweight", "dbias", "dfilm"), grads):
        assert torch.allclose(out[k], gr, atol=1e-11), k


def test_ctypes_descriptor_matches_the_header(tmp_path):
    """sizeof and the offsets of every field, as the C compiler lays them out."""
    import os
    import shutil
    import subprocess
    import common as C
    from ivid_amd import _lib
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    names = [n for n, _ in _lib.GnActDesc._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ivid_hip.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu\\n", offsetof(ivid_gn_act_desc, {n}));\n' for n in names)
                   + '  printf("%zu\\n", sizeof(ivid_gn_act_desc));\n  return 0;\n}\n')
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-I" + os.path.join(C.ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    assert got == [getattr(_lib.GnActDesc, n).offset for n in names] + [ctypes.sizeof(_lib.GnActDesc)]
