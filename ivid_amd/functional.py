"""Trainable operators of the UNet blocks, as autograd functions over the C ABI (include/ivid_hip.h ivid_gn_act_*, ivid_dropout).

    group_norm_act  GroupNorm32 -> FiLM -> SiLU -> Dropout of a ResBlock (adm.py:157-160,177-189,214-218) and the attention block's
                    norm (adm.py:274), in one pass over channels-last tensors, with the skip concat (adm.py:563) read in place
    dropout         nn.Dropout (adm.py:181) from a counter-based generator: no mask is stored

Both run on the tensors' device and on torch's current stream there, allocate through torch, never synchronise, and raise
IvidHipError for what the library refuses; wrong types, shapes and devices raise TypeError / ValueError before any launch.

`rng` of the dropout draws is (seed, stream_id), two integers in [0, 2^64), or an int64 tensor of those two on the device.  Equal
rng, equal draws: give every call of a step its own stream_id and every step its own seed.  The tensor form is read when the
kernels run, so that a captured graph draws anew once the host has rewritten it; the backward pass reads it again and must find
the forward's values (autograd's version check refuses a rewrite in between in eager code).

Capturing a training step into a graph: use the `*_forward` / `*_backward` pairs, which launch kernels and nothing else.  Under
capture the operators refuse tensors that require gradients, leaves or not, because accumulating into a leaf whose earlier eager
graph still lives would make the capturing stream wait for that graph's stream, which ends the process.  For the same reason do
not capture the backward pass of a graph that was built in eager code.

Forward-mode derivatives do not exist here: tensors that carry a tangent (torch.autograd.forward_ad) are refused.

Small training calls are bound by the host, and half of that is torch's change to its own thread for the backward pass: forward and
gradients of a 7 x 37 x 23 x 100 tensor take 130 us, 72 under torch.autograd.set_multithreading_enabled(False).
"""
import ctypes as C
import math

import torch
import torch.autograd.forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_ACTS = {"none": 0, "silu": 1}
_INT_MAX = (1 << 31) - 1
_MAX_POLLS = 0      # ivid_gn_act_desc.max_polls; the tests lower it


def _rng_args(rng, p, device):
    """(seed, stream_id, device pointer or None)"""
    if p == 0:
        return 0, 0, None
    if rng is None:
        raise ValueError("dropout with p > 0 needs rng = (seed, stream_id) or an int64 device tensor of the two")
    if isinstance(rng, torch.Tensor):
        if rng.dtype != torch.int64 or rng.shape != (2,) or not rng.is_contiguous() or rng.device != device:
            raise ValueError(f"rng must be a contiguous int64 tensor of 2 values on {device}")
        return 0, 0, rng.data_ptr()
    seed, stream_id = rng
    if not (0 <= seed < 1 << 64 and 0 <= stream_id < 1 << 64):
        raise ValueError("seed and stream_id must be in [0, 2^64)")
    return seed, stream_id, None


def _check_p(p):
    if not 0.0 <= p <= 1.0:     # refuses NaN too
        raise ValueError(f"dropout probability must be in [0, 1], got {p}")
    return float(p)


def _check_x(x, name):
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    if not x.is_cuda:
        raise _lib.IvidHipError(f"{name} is on {x.device}: ivid_amd has no CPU path")


_entry = {}     # the library's entry points by name


def _launch(name, device, *args):
    """One library call on torch's current stream of `device`, which is made current for it when it is not."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(_lib.load(), name)
    index = device.index
    # (the raw getters are torch.cuda.current_device() and torch.cuda.current_stream(index).cuda_stream without their 2 us)
    if index == torch._C._cuda_getDevice():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, name)


def _refuse_capture():
    if torch.cuda.is_current_stream_capturing():
        raise _lib.IvidHipError("autograd under graph capture: use the *_forward / *_backward functions, or no_grad "
                                "(see ivid_amd.functional)")


def _refuse_tangents(*tensors):
    """The kernels propagate none, and an output without one would read as a zero derivative.  (Outside of a level this costs 0.1 us.)"""
    if _forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        if any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
            raise _lib.IvidHipError("a tensor carries a forward-mode tangent: these operators have reverse-mode gradients only")


# ---- dropout ----
def _dropout(x, p, rng):
    if not x.is_contiguous():
        x = x.contiguous()
    out = torch.empty_like(x)
    n = x.numel()
    if n:
        device = x.device
        seed, sid, dev = _rng_args(rng, p, device)
        _launch("ivid_dropout", device, _DTYPES[x.dtype], x.data_ptr(), out.data_ptr(), n, p, seed, sid, dev)
    return out


# The backward passes run in autograd's own thread, where Python is several times slower than in the caller's: what can be prepared in
# the forward call is, and the wrapper that makes them differentiable once is only entered under create_graph.
def _dropout_grads(ctx, dy):
    if _forward_ad._current_level >= 0:
        _refuse_tangents(dy)
    return _dropout(dy, ctx.p, ctx.saved_tensors[0] if ctx.device_rng else ctx.rng), None, None


_dropout_grads_once = once_differentiable(_dropout_grads)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng):
        y = _dropout(x, p, rng)
        ctx.p, ctx.device_rng = p, isinstance(rng, torch.Tensor)
        if ctx.device_rng:
            ctx.save_for_backward(rng)
        else:      # (the caller may rewrite a list; without draws rng may be anything)
            ctx.rng = tuple(rng) if p and y.numel() else None
        return y

    @staticmethod
    def backward(ctx, dy):
        return _dropout_grads_once(ctx, dy) if torch.is_grad_enabled() else _dropout_grads(ctx, dy)


def dropout(x, p, rng=None):
    """y[i] = x[i] * 65536 / (65536 - T) where draw(i) >= T = floor(p * 65536 + 1/2), else 0; i = the row-major index.

    x any shape, float32 / bfloat16 / float16; other than contiguous tensors are copied first.  The draws are a function of (rng, i)
    alone (include/ivid_hip.h ivid_dropout); a dropped element is 0 whatever x holds.  p is used in steps of 2^-16: below 2^-17 it
    copies, from 1 - 2^-17 on it drops all; p = 0 needs no rng.  Under capture, and for the gradient by hand, call it on the gradient
    with the same rng: the operator is its own backward pass."""
    _check_x(x, "x")
    p = _check_p(p)
    _refuse_tangents(x)
    if torch.is_grad_enabled() and x.requires_grad:
        _refuse_capture()
        return _Dropout.apply(x, p, rng)
    return _dropout(x, p, rng)


# ---- GroupNorm + FiLM + activation + dropout ----
def _pixels(x):
    """x [N, ..., C] as (tensor, pixel stride, sample stride): in place when the channels are contiguous and the inner dimensions
    collapse to one stride, else a contiguous copy."""
    n, c = x.shape[0], x.shape[-1]
    hw = x.numel() // (n * c) if n and c else 0
    if x.is_contiguous():
        return x, c, hw * c
    if x.stride(-1) == 1 or c == 1:
        ld, size = None, 1
        for d in range(x.dim() - 2, 0, -1):
            if x.shape[d] == 1:
                continue
            if ld is None:
                ld = x.stride(d)
            elif x.stride(d) != ld * size:
                break
            size *= x.shape[d]
        else:
            return x, c if ld is None else ld, x.stride(0)
    x = x.contiguous()
    return x, c, hw * c


class _Call:
    """Checked arguments of one group_norm_act call, as the library takes them."""

    def __init__(self, x, groups, weight, bias, film, skip, act, eps, p, rng):
        _check_x(x, "x")
        dev, dtype, shape = x.device, x.dtype, x.shape
        if len(shape) < 2:
            raise ValueError("x must be [N, ..., C]")
        n, c0, c1 = shape[0], shape[-1], 0
        if skip is not None:
            if skip.dtype != dtype or skip.device != dev or skip.shape[:-1] != shape[:-1]:
                raise ValueError("skip must match x in everything but the number of channels")
            c1 = skip.shape[-1]
        c = c0 + c1
        if c0 == 0 or (skip is not None and c1 == 0):
            raise ValueError("x and skip need channels")
        if groups <= 0 or c % groups:
            raise ValueError(f"{c} channels are not divisible by {groups} groups")
        for name, t in (("weight", weight), ("bias", bias)):
            if t.dtype != torch.float32:
                raise TypeError(f"{name} must be float32, got {t.dtype}")
            if t.dim() != 1 or t.shape[0] != c or t.device != dev:
                raise ValueError(f"{name} must be [{c}] on {dev}")
        if film is not None:
            if film.dtype != torch.float32 and film.dtype != dtype:
                raise TypeError(f"film must be float32 or {dtype}, got {film.dtype}")
            if film.shape != (n, 2 * c) or film.device != dev:
                raise ValueError(f"film must be [{n}, {2 * c}] (scale, shift) on {dev}")
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}, got {act!r}")
        if not (eps > 0 and math.isfinite(eps)):
            raise ValueError(f"eps must be positive, got {eps}")
        p = _check_p(p)
        numel = x.numel()
        hw = numel // (n * c0) if numel else 0
        if max(n, hw, c) > _INT_MAX:      # the descriptor's ints would wrap without a word
            raise ValueError(f"[{n}, {hw}, {c}] is too large: every size must be below 2^31")
        self.device, self.index, self.dtype = dev, x.get_device(), dtype
        if film is not None:
            self.film_shape, self.film_dtype = film.shape, film.dtype
        if c1:
            self.skip_shape = skip.shape
        self.shape = shape if c1 == 0 else shape[:-1] + (c,)
        self.x_shape, self.c_shape, self.stats_shape = shape, (c,), (n, groups, 2)
        self.n, self.c0, self.c1, self.c, self.groups, self.p = n, c0, c1, c, groups, p
        self.empty = numel == 0
        d = self.desc = _lib.GnActDesc(_DTYPES[dtype], n, hw, c0, c1, groups, _ACTS[act])
        d.eps, d.p, d.max_polls = eps, p, _MAX_POLLS
        self.bind(x, weight, bias, film, skip, rng)

    def bind(self, x, weight, bias, film, skip, rng):
        """Point the descriptor at these tensors (of the shapes and types checked in front), which the caller keeps alive."""
        d = self.desc
        self.in_place = (x.is_contiguous() and weight.is_contiguous() and bias.is_contiguous()
                         and (film is None or film.is_contiguous()) and (skip is None or skip.is_contiguous()))
        x, d.ld0, d.sn0 = _pixels(x)
        if skip is not None:
            skip, d.ld1, d.sn1 = _pixels(skip)
        weight, bias = weight.contiguous(), bias.contiguous()
        if film is not None:
            if film.stride(1) != 1:
                film = film.contiguous()
            d.film_ld, d.film_dtype = film.stride(0), _DTYPES[film.dtype]
        self.point((x.data_ptr(), None if skip is None else skip.data_ptr(), weight.data_ptr(), bias.data_ptr(),
                    None if film is None else film.data_ptr()))
        d.seed, d.stream_id, d.rng = _rng_args(rng, self.p, self.device)
        self.device_rng = d.rng is not None
        self.keep = (x, skip, weight, bias, film, rng)

    def point(self, at):
        d = self.desc
        self.at = d.src0, d.src1, d.gamma, d.beta, d.film = at
        self.backward_bytes = None      # depends on strides and alignment

    def rebind(self, x, weight, bias, film, skip, rng):
        """bind() for the tensors that autograd saved, which are mostly where they were.  A hook may unpack others."""
        index = self.index
        same = (x.shape == self.x_shape and x.dtype is self.dtype and x.get_device() == index
                and weight.shape == bias.shape == self.c_shape and weight.dtype is bias.dtype is torch.float32
                and weight.get_device() == bias.get_device() == index)
        if film is not None:
            same = same and film.shape == self.film_shape and film.dtype is self.film_dtype and film.get_device() == index
        if skip is not None:
            same = same and skip.shape == self.skip_shape and skip.dtype is self.dtype and skip.get_device() == index
        if not same:      # the launch would read past its end
            raise ValueError("a saved tensor came back with another type, shape or device")
        if self.in_place and (x.is_contiguous() and weight.is_contiguous() and bias.is_contiguous()
                              and (film is None or film.is_contiguous()) and (skip is None or skip.is_contiguous())):
            at = (x.data_ptr(), None if skip is None else skip.data_ptr(), weight.data_ptr(), bias.data_ptr(),
                  None if film is None else film.data_ptr())
            if at != self.at:
                self.point(at)
            if self.device_rng:
                self.desc.rng = _rng_args(rng, self.p, self.device)[2]
        else:
            self.bind(x, weight, bias, film, skip, rng)

    def scratch_bytes(self, backward):
        fn = _entry.get("scratch")
        if fn is None:
            fn = _entry["scratch"] = _lib.load().ivid_gn_act_scratch_bytes
        nbytes = fn(C.byref(self.desc), backward)
        if nbytes < 0:
            _lib.check(-1, "ivid_gn_act_scratch_bytes")
        return nbytes

    def scratch(self, backward):
        nbytes = self.backward_bytes if backward and self.backward_bytes is not None else self.scratch_bytes(backward)
        if nbytes == 0:
            return None, 0, None
        buf = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        return buf.data_ptr(), nbytes, buf

    def forward(self):
        y = torch.empty(self.shape, dtype=self.dtype, device=self.device)
        stats = torch.empty(self.stats_shape, dtype=torch.float32, device=self.device)
        if self.empty:
            return y, stats.zero_()
        ptr, nbytes, buf = self.scratch(0)
        _launch("ivid_gn_act_forward", self.device, C.byref(self.desc), y.data_ptr(), stats.data_ptr(), ptr, nbytes)
        return y, stats

    def check_gradient(self, dy):
        if dy.shape != self.shape or dy.dtype != self.dtype or dy.device != self.device:
            raise ValueError(f"dy must be {tuple(self.shape)} {self.dtype} on {self.device}")

    def backward(self, dy, stats):
        self.check_gradient(dy)
        x, skip, weight, bias, film, _ = self.keep
        return self.gradients(dy, stats, x, weight, bias, film, skip)

    def gradients(self, dy, stats, x, weight, bias, film, skip):
        if stats.shape != self.stats_shape or stats.dtype is not torch.float32 or stats.get_device() != self.index:
            raise ValueError("stats must be what the forward call returned")
        if not stats.is_contiguous():
            stats = stats.contiguous()
        if not dy.is_contiguous():
            dy = dy.contiguous()
        if dy.data_ptr() % 16:
            dy = dy.clone()
        dev = self.device
        dskip = dfilm = None
        if self.in_place and not self.empty:
            like = torch.empty_like
            dx, dweight, dbias = like(x), like(weight), like(bias)
            if skip is not None:
                dskip = like(skip)
            if film is not None:
                dfilm = like(film)
        else:
            new = torch.zeros if self.empty else torch.empty
            dx = new(self.shape[:-1] + (self.c0,), dtype=self.dtype, device=dev)
            dweight = new(self.c, dtype=torch.float32, device=dev)
            dbias = new(self.c, dtype=torch.float32, device=dev)
            if skip is not None:
                dskip = new(self.shape[:-1] + (self.c1,), dtype=self.dtype, device=dev)
            if film is not None:
                dfilm = new((self.n, 2 * self.c), dtype=self.film_dtype, device=dev)
            if self.empty:
                return dx, dskip, dweight, dbias, dfilm
        ptr, nbytes, buf = self.scratch(1)
        _launch("ivid_gn_act_backward", dev, C.byref(self.desc), stats.data_ptr(), dy.data_ptr(), dx.data_ptr(),
                None if dskip is None else dskip.data_ptr(), dweight.data_ptr(), dbias.data_ptr(),
                None if dfilm is None else dfilm.data_ptr(), ptr, nbytes)
        return dx, dskip, dweight, dbias, dfilm


def _gn_grads(ctx, dy):
    if _forward_ad._current_level >= 0:
        _refuse_tangents(dy)
    x, weight, bias, film, skip, stats, rng = ctx.saved_tensors
    if rng is None:
        rng = ctx.rng
    try:
        call = ctx.calls.pop()      # (one step under the interpreter's lock: threads may walk one retained graph at once)
    except IndexError:
        groups, act, eps, p = ctx.args
        call = _Call(x, groups, weight, bias, film, skip, act, eps, p, rng)
        call.check_gradient(dy)
    else:
        call.rebind(x, weight, bias, film, skip, rng)
    dx, dskip, dw, db, dfilm = call.gradients(dy, stats, x, weight, bias, film, skip)
    call.keep = None
    ctx.calls.append(call)
    need = ctx.needs_input_grad
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, dfilm if need[3] else None,
            dskip if need[4] else None, None, None, None, None, None)


_gn_grads_once = once_differentiable(_gn_grads)


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, film, skip, groups, act, eps, p, rng):
        call = _Call(x, groups, weight, bias, film, skip, act, eps, p, rng)
        y, stats = call.forward()
        device_rng = isinstance(rng, torch.Tensor)
        ctx.save_for_backward(x, weight, bias, film, skip, stats, rng if device_rng else None)
        call.keep = None        # what saves, offloads or recomputes saved tensors decides over their lives
        if not call.empty:
            call.backward_bytes = call.scratch_bytes(1)
        ctx.calls, ctx.args = [call], (groups, act, eps, p)
        ctx.rng = tuple(rng) if p and not device_rng else None      # (the caller may rewrite a list)
        return y

    @staticmethod
    def backward(ctx, dy):
        return _gn_grads_once(ctx, dy) if torch.is_grad_enabled() else _gn_grads(ctx, dy)


def group_norm_act(x, groups, weight, bias, film=None, skip=None, act="silu", eps=1e-5, p=0.0, rng=None):
    """y = drop(act(u * (1 + scale) + shift)), u = (x - mean) * rstd * weight + bias, statistics per sample and group.

    x        [N, ..., C0], float32 / bfloat16 / float16, channels last (a torch channels_last NCHW tensor: x.permute(0, 2, 3, 1)); read in
             place when its channels are contiguous and its pixels have one stride, else copied first
    skip     [N, ..., C1]: channels concatenated behind x's, never materialised (adm.py:563); C = C0 + C1
    weight, bias   float32 [C]
    film     [N, 2C] float32 or x's type, scale then shift (adm.py:214-218); rows may be strided; None: no FiLM
    act      "silu" or "none"
    p, rng   dropout of the result, as `dropout` with the index in the [N, ..., C] output
    Returns [N, ..., C] of x's type; statistics, sums and the arithmetic are 32 bits or wider whatever x's type, the result is rounded
    once.  Differentiable once in x, skip, weight, bias and film."""
    _refuse_tangents(x, skip, weight, bias, film)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, film, skip)):
        _refuse_capture()
        return _GroupNormAct.apply(x, weight, bias, film, skip, groups, act, eps, p, rng)
    return _Call(x, groups, weight, bias, film, skip, act, eps, p, rng).forward()[0]


@torch.no_grad()
def group_norm_act_forward(x, groups, weight, bias, film=None, skip=None, act="silu", eps=1e-5, p=0.0, rng=None):
    """group_norm_act without autograd: (y, stats), stats fp32 [N, groups, 2] = mean, rstd."""
    _refuse_tangents(x, skip, weight, bias, film)
    return _Call(x, groups, weight, bias, film, skip, act, eps, p, rng).forward()


@torch.no_grad()
def group_norm_act_backward(dy, stats, x, groups, weight, bias, film=None, skip=None, act="silu", eps=1e-5, p=0.0, rng=None):
    """Gradients (dx, dskip, dweight, dbias, dfilm; None where there is no input) of the group_norm_act_forward call with these
    arguments that returned `stats`."""
    _refuse_tangents(dy, stats, x, skip, weight, bias, film)
    return _Call(x, groups, weight, bias, film, skip, act, eps, p, rng).backward(dy, stats)
