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
capture the autograd forms are refused for leaves that require gradients, because accumulating into a leaf whose earlier eager
graph still lives would make the capturing stream wait for that graph's stream, which ends the process.
"""
import ctypes as C
import math

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_ACTS = {"none": 0, "silu": 1}
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


class _on:
    """The tensors' device made current for the launches, when it is not."""

    def __init__(self, device):
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard:
            self.guard.__exit__(*exc)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _refuse_captured_leaves(*tensors):
    if torch.cuda.is_current_stream_capturing() and any(t is not None and t.requires_grad and t.is_leaf for t in tensors):
        raise _lib.IvidHipError("autograd through a leaf under graph capture: use the *_forward / *_backward functions "
                                "(see ivid_amd.functional)")


# ---- dropout ----
def _dropout(x, p, rng):
    x = x.contiguous()
    out = torch.empty_like(x)
    if x.numel():
        seed, sid, dev = _rng_args(rng, p, x.device)
        with _on(x.device):
            _lib.call("ivid_dropout", _DTYPES[x.dtype], x.data_ptr(), out.data_ptr(), x.numel(), p, seed, sid, dev,
                      _stream(x.device))
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng):
        ctx.p, ctx.rng = p, rng
        if isinstance(rng, torch.Tensor):
            ctx.save_for_backward(rng)
            ctx.rng = None
        return _dropout(x, p, rng)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return _dropout(dy, ctx.p, ctx.saved_tensors[0] if ctx.saved_tensors else ctx.rng), None, None


def dropout(x, p, rng=None):
    """y[i] = x[i] * 65536 / (65536 - T) where draw(i) >= T = floor(p * 65536 + 1/2), else 0; i = the row-major index.

    x any shape, float32 / bfloat16 / float16; other than contiguous tensors are copied first.  The draws are a function of (rng, i)
    alone (include/ivid_hip.h ivid_dropout); a dropped element is 0 whatever x holds; p = 0 copies.  Under capture, and for the
    gradient by hand, call it on the gradient with the same rng: the operator is its own backward pass."""
    _check_x(x, "x")
    p = _check_p(p)
    _rng_args(rng, p, x.device)
    if torch.is_grad_enabled() and x.requires_grad:
        _refuse_captured_leaves(x)
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
    """Checked arguments of one group_norm_act call, as the library takes them; keeps what the descriptor points to alive."""

    def __init__(self, x, groups, weight, bias, film, skip, act, eps, p, rng):
        _check_x(x, "x")
        if x.dim() < 2:
            raise ValueError("x must be [N, ..., C]")
        n, c0 = x.shape[0], x.shape[-1]
        c1 = 0
        dev = x.device
        if skip is not None:
            if skip.dtype != x.dtype or skip.device != dev or skip.shape[:-1] != x.shape[:-1]:
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
            if t.shape != (c,) or t.device != dev:
                raise ValueError(f"{name} must be [{c}] on {dev}")
        if film is not None:
            if film.dtype not in (torch.float32, x.dtype):
                raise TypeError(f"film must be float32 or {x.dtype}, got {film.dtype}")
            if film.shape != (n, 2 * c) or film.device != dev:
                raise ValueError(f"film must be [{n}, {2 * c}] (scale, shift) on {dev}")
            if film.stride(1) != 1:
                film = film.contiguous()
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}, got {act!r}")
        if not (eps > 0 and math.isfinite(eps)):
            raise ValueError(f"eps must be positive, got {eps}")
        p = _check_p(p)
        seed, sid, rng_ptr = _rng_args(rng, p, dev)
        self.shape = x.shape[:-1] + (c,)
        self.device, self.dtype = dev, x.dtype
        self.n, self.c0, self.c1, self.c, self.groups = n, c0, c1, c, groups
        self.empty = x.numel() == 0
        x, ld0, sn0 = _pixels(x)
        if skip is not None:
            skip, ld1, sn1 = _pixels(skip)
        else:
            ld1 = sn1 = 0
        weight, bias = weight.contiguous(), bias.contiguous()
        self.keep = (x, skip, weight, bias, film, rng)
        ptr = _lib.ptr
        self.film = film
        self.desc = _lib.GnActDesc(
            _DTYPES[x.dtype], n, 0 if self.empty else x.numel() // (n * c0), c0, c1, groups, _ACTS[act],
            x.data_ptr(), ld0, sn0, ptr(skip), ld1, sn1, weight.data_ptr(), bias.data_ptr(), ptr(film),
            _DTYPES[film.dtype] if film is not None else 0, film.stride(0) if film is not None else 0, eps, p, seed, sid, rng_ptr,
            _MAX_POLLS)

    def scratch(self, backward):
        nbytes = _lib.load().ivid_gn_act_scratch_bytes(C.byref(self.desc), backward)
        if nbytes < 0:
            _lib.check(-1, "ivid_gn_act_scratch_bytes")
        return (torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None), nbytes

    def forward(self):
        y = torch.empty(self.shape, dtype=self.dtype, device=self.device)
        stats = torch.empty(self.n, self.groups, 2, dtype=torch.float32, device=self.device)
        if self.empty:
            return y, stats.zero_()
        with _on(self.device):
            scratch, nbytes = self.scratch(0)
            _lib.call("ivid_gn_act_forward", C.byref(self.desc), y.data_ptr(), stats.data_ptr(), _lib.ptr(scratch), nbytes,
                      _stream(self.device))
        return y, stats

    def backward(self, dy, stats):
        if dy.shape != self.shape or dy.dtype != self.dtype or dy.device != self.device:
            raise ValueError(f"dy must be {tuple(self.shape)} {self.dtype} on {self.device}")
        if stats.shape != (self.n, self.groups, 2) or stats.dtype != torch.float32 or stats.device != self.device:
            raise ValueError("stats must be what the forward call returned")
        dy, stats = dy.contiguous(), stats.contiguous()
        if dy.data_ptr() % 16:
            dy = dy.clone()
        new = torch.zeros if self.empty else torch.empty
        dev = self.device
        dx = new(self.shape[:-1] + (self.c0,), dtype=self.dtype, device=dev)
        dskip = new(self.shape[:-1] + (self.c1,), dtype=self.dtype, device=dev) if self.c1 else None
        dparam = new(2, self.c, dtype=torch.float32, device=dev)
        dfilm = new(self.n, 2 * self.c, dtype=self.film.dtype, device=dev) if self.film is not None else None
        if not self.empty:
            with _on(dev):
                scratch, nbytes = self.scratch(1)
                _lib.call("ivid_gn_act_backward", C.byref(self.desc), stats.data_ptr(), dy.data_ptr(), dx.data_ptr(), _lib.ptr(dskip),
                          dparam.data_ptr(), dparam.data_ptr() + 4 * self.c, _lib.ptr(dfilm), _lib.ptr(scratch), nbytes, _stream(dev))
        return dx, dskip, dparam[0], dparam[1], dfilm


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, film, skip, groups, act, eps, p, rng):
        call = _Call(x, groups, weight, bias, film, skip, act, eps, p, rng)
        y, stats = call.forward()
        ctx.save_for_backward(x, weight, bias, film, skip, stats, rng if isinstance(rng, torch.Tensor) else None)
        ctx.args = (groups, act, eps, p, rng if not isinstance(rng, torch.Tensor) else None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, film, skip, stats, rng_t = ctx.saved_tensors
        groups, act, eps, p, rng = ctx.args
        call = _Call(x, groups, weight, bias, film, skip, act, eps, p, rng_t if rng_t is not None else rng)
        dx, dskip, dw, db, dfilm = call.backward(dy, stats)
        need = ctx.needs_input_grad
        return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, dfilm if need[3] else None,
                dskip if need[4] else None, None, None, None, None, None)


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
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, film, skip)):
        _refuse_captured_leaves(x, weight, bias, film, skip)
        return _GroupNormAct.apply(x, weight, bias, film, skip, groups, act, eps, p, rng)
    return _Call(x, groups, weight, bias, film, skip, act, eps, p, rng).forward()[0]


@torch.no_grad()
def group_norm_act_forward(x, groups, weight, bias, film=None, skip=None, act="silu", eps=1e-5, p=0.0, rng=None):
    """group_norm_act without autograd: (y, stats), stats fp32 [N, groups, 2] = mean, rstd."""
    return _Call(x, groups, weight, bias, film, skip, act, eps, p, rng).forward()


@torch.no_grad()
def group_norm_act_backward(dy, stats, x, groups, weight, bias, film=None, skip=None, act="silu", eps=1e-5, p=0.0, rng=None):
    """Gradients (dx, dskip, dweight, dbias, dfilm; None where there is no input) of the group_norm_act_forward call with these
    arguments that returned `stats`."""
    return _Call(x, groups, weight, bias, film, skip, act, eps, p, rng).backward(dy, stats)
