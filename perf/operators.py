"""Workloads of the trainable UNet operators, for measuring them: GroupNorm with FiLM, activation and dropout over
channels-last tensors, and dropout from a counter-based generator whose mask is never stored.

A case is run either in plain form (`own` false: elementary torch operations in 32 bits, rounded once at the end) or through
`ivid_amd.functional` (`own` true).

    y = drop(act(((x - mean) * rstd * weight + bias) * (1 + scale) + shift))

x [N, ..., C] (C = the channels of `x` followed by those of `skip`, the skip concatenation of a decoder block), mean and variance
per sample and group of C / groups channels; scale | shift = the halves of film [N, 2C].  Element i (row-major) of a dropped
tensor is kept when its 16-bit draw is >= T = floor(p * 65536 + 1/2), and then multiplied by 65536 / (65536 - T).  Draw i is half
i % 2 (low half first) of word (i % 8) / 2 of the Philox4x32-10 block with counter (i / 8, stream) and key seed ^ (DROP << 32).
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DROP = 0x44524F50
M32 = 0xFFFFFFFF


def gn(name, n, hw, c, dtype, direction, groups=32, c_skip=0, film=False, act="silu", p=0.0):
    return {"name": name, "op": "gn", "n": n, "h": hw[0], "w": hw[1], "c": c, "c_skip": c_skip, "groups": groups, "dtype": dtype,
            "direction": direction, "film": film, "act": act, "p": p}


def drop(name, numel, dtype, direction, p):
    return {"name": name, "op": "dropout", "numel": numel, "dtype": dtype, "direction": direction, "p": p}


def listed():
    """Widths, resolutions and batch are those of the 128 x 128 backbones (256 or 128 base channels, multipliers 1 1 2 3 4,
    32 groups, batch 64); the odd ones stand for images and widths nobody tuned for."""
    return [
        # one sample at the bottleneck: nothing but latency
        gn("gn_fwd_b1_8x8_c1024_fp16", 1, (8, 8), 1024, "fp16", "forward"),
        # the second norm of a ResBlock in evaluation, with FiLM, at the 16 x 16 level
        gn("gn_fwd_b64_16x16_c768_bf16_film", 64, (16, 16), 768, "bf16", "forward", film=True),
        # the same at the first level: the largest tensor of the network
        gn("gn_fwd_b64_128x128_c256_bf16_film", 64, (128, 128), 256, "bf16", "forward", film=True),
        # a training step's second norm: FiLM, SiLU and dropout in front of the second convolution
        gn("gn_train_b64_32x32_c512_bf16_film_drop", 64, (32, 32), 512, "bf16", "train", film=True, p=0.1),
        # ... and at the first level, the largest
        gn("gn_train_b64_128x128_c256_bf16_film_drop", 64, (128, 128), 256, "bf16", "train", film=True, p=0.1),
        # a decoder block's first norm reads the skip concatenation (56 channels a group, one group across the seam)
        gn("gn_train_b64_16x16_c1024_skip768_fp16", 64, (16, 16), 1024, "fp16", "train", c_skip=768),
        # the norm of an attention block: no activation, one sample is a sequence of 1024 pixels
        gn("gn_train_b32_seq1024_c512_bf16_noact", 32, (1024, 1), 512, "bf16", "train", act="none"),
        # the small backbone in full precision
        gn("gn_train_b16_64x64_c128_fp32_film", 16, (64, 64), 128, "fp32", "train", film=True),
        # odd everything: 5 channels a group, 200-byte pixels, a pixel count that divides by nothing
        gn("gn_train_b7_37x23_c100_g20_fp16_drop", 7, (37, 23), 100, "fp16", "train", groups=20, film=True, p=0.25),
        # dropout of an embedding: latency
        drop("dropout_fwd_64x1024_fp32", 64 * 1024, "fp32", "forward", 0.1),
        # a length that is no multiple of anything
        drop("dropout_train_1000003_fp16", 1000003, "fp16", "train", 0.3),
        # the largest activation of the network
        drop("dropout_train_b64_128x128_c256_bf16", 64 * 128 * 128 * 256, "bf16", "train", 0.1),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(sorted(DTYPES))
    direction = rng.choice(["forward", "train"])
    if rng.random() < 0.25:
        return drop(None, log_int(rng, 1000, 1 << 27), dtype, direction, rng.choice([0.05, 0.1, 0.3, 0.5]))
    groups = rng.choice([1, 2, 4, 8, 16, 20, 32, 32, 32])
    h, w = log_int(rng, 1, 128), log_int(rng, 1, 128)
    cg = log_int(rng, 1, 2048 // groups if groups > 2 else 256)
    c = groups * max(cg, 8 // (h * w))      # eight values a group at least: fewer have no variance to speak of
    c_skip = 0
    if rng.random() < 0.25 and c >= 64:
        c_skip = (c // rng.choice([2, 3, 4])) & ~7
    most = 1 << 27      # elements; the largest listed case has twice that
    n = log_int(rng, 1, 64)
    n = max(1, min(n, most // (h * w * c)))
    return gn(None, n, (h, w), c - c_skip, dtype, direction, groups=groups, c_skip=c_skip, film=rng.random() < 0.5,
              act=rng.choice(["silu", "silu", "none"]), p=rng.choice([0.0, 0.0, 0.1, 0.3]))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 12345)
    dt = DTYPES[case["dtype"]]
    train = case["direction"] == "train"
    rng = ((seed * 0x9E3779B97F4A7C15 + 0x1234567) & 0x7FFFFFFFFFFFFFFF, seed % 1000 + 1)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["op"] == "dropout":
        s = {"case": case, "rng": rng, "x": randn(case["numel"]).to(dt)}
        if train:
            s["x"].requires_grad_()
            s["dy"] = randn(case["numel"]).to(dt)
        return s
    n, h, w, c0, c1 = case["n"], case["h"], case["w"], case["c"], case["c_skip"]
    c = c0 + c1

    def activation(ch):      # channels differ in mean and spread, as convolution outputs do
        x = randn(n, h, w, ch)
        x *= 0.5 + torch.rand(ch, generator=g, device=dev)
        x += 0.5 * randn(ch)
        return x.to(dt)

    s = {"case": case, "rng": rng, "x": activation(c0), "skip": activation(c1) if c1 else None,
         "weight": 1.0 + 0.2 * randn(c), "bias": 0.2 * randn(c), "film": 0.3 * randn(n, 2 * c) if case["film"] else None}
    if train:
        s["dy"] = randn(n, h, w, c).to(dt)
        for k in ("x", "skip", "weight", "bias", "film"):
            if s[k] is not None:
                s[k].requires_grad_()
    return s


# ---- plain form ----
def philox(counter, stream, key):
    """Philox4x32-10 over int64 tensors that hold 32-bit words (the low and high half of a 64-bit product that wraps are right)."""
    k0, k1 = key & M32, key >> 32
    c = [counter & M32, counter >> 32, torch.full_like(counter, stream & M32), torch.full_like(counter, stream >> 32)]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & M32) ^ c[1] ^ k0, b & M32, ((a >> 32) & M32) ^ c[3] ^ k1, a & M32]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return c


def threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def kept(numel, p, rng, device):
    blocks = torch.arange((numel + 7) // 8, device=device)
    words = torch.stack(philox(blocks, rng[1], rng[0] ^ (DROP << 32)), -1)
    draws = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:numel]
    return draws >= threshold(p)


def plain_dropout(x, keep, p):
    t = threshold(p)
    return torch.where(keep, x * (65536.0 / (65536 - t) if t < 65536 else 0.0), 0.0)


def plain_gn(s):
    case = s["case"]
    x = s["x"].detach().float()
    if s["skip"] is not None:
        x = torch.cat([x, s["skip"].detach().float()], -1)
    n, h, w, c = x.shape
    grp = case["groups"]
    dt = DTYPES[case["dtype"]]
    xg = x.reshape(n, h * w, grp, c // grp)
    mean = xg.mean((1, 3), keepdim=True)
    xc = xg - mean
    rstd = torch.rsqrt((xc * xc).mean((1, 3), keepdim=True) + 1e-5)
    xhat = (xc * rstd).reshape(n, h * w, c)
    gamma, beta = s["weight"].detach(), s["bias"].detach()
    u = xhat * gamma + beta
    v = u
    if s["film"] is not None:
        film = s["film"].detach().float()
        gain = 1.0 + film[:, None, :c]
        v = u * gain + film[:, None, c:]
    sig = torch.sigmoid(v) if case["act"] == "silu" else None
    y = v * sig if sig is not None else v
    keep = kept(y.numel(), case["p"], s["rng"], y.device).reshape(y.shape) if case["p"] > 0 else None
    if keep is not None:
        y = plain_dropout(y, keep, case["p"])
    out = {"y": y.reshape(n, h, w, c).to(dt)}
    if case["direction"] == "forward":
        return out
    gv = s["dy"].float().reshape(n, h * w, c)
    if keep is not None:
        gv = plain_dropout(gv, keep, case["p"])
    if sig is not None:
        gv = gv * (sig * (1.0 + v * (1.0 - sig)))
    gu = gv * gain if s["film"] is not None else gv
    gx = (gu * gamma).reshape(n, h * w, grp, c // grp)
    xhg = xhat.reshape(n, h * w, grp, c // grp)
    dx = rstd * (gx - gx.mean((1, 3), keepdim=True) - xhg * (gx * xhg).mean((1, 3), keepdim=True))
    dx = dx.reshape(n, h, w, c)
    out["dx"] = dx[..., :case["c"]].to(dt)
    if s["skip"] is not None:
        out["dskip"] = dx[..., case["c"]:].to(dt)
    out["dweight"] = (gu * xhat).sum((0, 1))
    out["dbias"] = gu.sum((0, 1))
    if s["film"] is not None:
        out["dfilm"] = torch.cat([(gv * u).sum(1), gv.sum(1)], 1)
    return out


def run(state):
    case = state["case"]
    train = case["direction"] == "train"
    if own:
        from ivid_amd import functional as F
        if case["op"] == "dropout":
            y = F.dropout(state["x"], case["p"], state["rng"])
            return {"y": y, "dx": torch.autograd.grad(y, state["x"], state["dy"])[0]} if train else {"y": y}
        y = F.group_norm_act(state["x"], case["groups"], state["weight"], state["bias"], film=state["film"], skip=state["skip"],
                             act=case["act"], p=case["p"], rng=state["rng"] if case["p"] > 0 else None)
        if not train:
            return {"y": y}
        names = [k for k in ("x", "skip", "weight", "bias", "film") if state[k] is not None]
        grads = torch.autograd.grad(y, [state[k] for k in names], state["dy"])
        return dict({"y": y.detach()}, **{"d" + k: g for k, g in zip(names, grads)})
    with torch.no_grad():
        if case["op"] == "dropout":
            keep = kept(case["numel"], case["p"], state["rng"], state["x"].device)
            out = {"y": plain_dropout(state["x"].float(), keep, case["p"]).to(state["x"].dtype)}
            if train:
                out["dx"] = plain_dropout(state["dy"].float(), keep, case["p"]).to(state["x"].dtype)
            return out
        return plain_gn(state)


def work(case):
    """Each input read once, each output written once.  Operations: 14 a normalised and activated element forward, 30 more backward,
    and the generator's 25 a draw (ten rounds of two products over eight elements)."""
    e = 4 if case["dtype"] == "fp32" else 2
    train = case["direction"] == "train"
    if case["op"] == "dropout":
        n = case["numel"]
        return {"bytes": n * e * (4 if train else 2), "flops": n * 27 * (2 if train else 1)}
    c = case["c"] + case["c_skip"]
    n = case["n"] * case["h"] * case["w"] * c
    small = 4 * (2 * c + (2 * case["n"] * c if case["film"] else 0))
    draws = 25 * n if case["p"] > 0 else 0
    if train:
        return {"bytes": 4 * n * e + 2 * small, "flops": 44 * n + 2 * draws}
    return {"bytes": 2 * n * e + small, "flops": 14 * n + draws}


# ---- the definition in 64 bits, sample by sample, gradients by automatic differentiation ----
def _mul_hi_lo(a, m):
    """High and low 32 bits of a * m, 0 <= a, m < 2^32, from 16-bit halves: no product passes 2^48."""
    lo16, hi16 = a * (m & 0xFFFF), a * (m >> 16)
    mid = lo16 // 65536 + hi16
    return mid // 65536, (mid % 65536) * 65536 + lo16 % 65536


def _draws(first, count, rng, device):
    """Draws first .. first + count - 1 of the stream."""
    b0 = first // 8
    b1 = (first + count + 7) // 8
    x0 = torch.arange(b0, b1, dtype=torch.int64, device=device)
    x1, x2, x3 = x0 // 2**32, torch.full_like(x0, rng[1] % 2**32), torch.full_like(x0, rng[1] // 2**32)
    x0 = x0 % 2**32
    ka, kb = rng[0] % 2**32, (rng[0] // 2**32) ^ DROP
    for _ in range(10):
        h0, l0 = _mul_hi_lo(x0, 0xD2511F53)
        h1, l1 = _mul_hi_lo(x2, 0xCD9E8D57)
        x0, x1, x2, x3 = h1 ^ x1 ^ ka, l1, h0 ^ x3 ^ kb, l0
        ka, kb = (ka + 0x9E3779B9) % 2**32, (kb + 0xBB67AE85) % 2**32
    out = torch.empty(b1 - b0, 8, dtype=torch.int64, device=device)
    for i, word in enumerate((x0, x1, x2, x3)):
        out[:, 2 * i] = word % 65536
        out[:, 2 * i + 1] = word // 65536
    return out.reshape(-1)[first - 8 * b0:first - 8 * b0 + count]


def exact(case, seed):
    s = prepare(case, seed)
    train = case["direction"] == "train"
    cut = math.floor(case["p"] * 65536 + 0.5)
    factor = 65536 / (65536 - cut)
    if case["op"] == "dropout":
        out = {k: torch.empty(case["numel"], dtype=torch.float64, device="cuda") for k in (("y", "dx") if train else ("y",))}
        step = 1 << 25
        for i in range(0, case["numel"], step):
            j = min(i + step, case["numel"])
            scale = (_draws(i, j - i, s["rng"], "cuda") >= cut).double() * factor
            out["y"][i:j] = s["x"].detach()[i:j].double() * scale
            if train:
                out["dx"][i:j] = s["dy"][i:j].double() * scale
        return out
    c, per = case["c"] + case["c_skip"], case["h"] * case["w"]
    rows = {k: [] for k in ("y", "dx", "dskip", "dfilm")}
    wt = s["weight"].detach().double().requires_grad_()
    bs = s["bias"].detach().double().requires_grad_()
    dwt, dbs = torch.zeros_like(wt), torch.zeros_like(bs)
    for i in range(case["n"]):
        leaves = {"x": s["x"][i].detach().double().requires_grad_()}
        if s["skip"] is not None:
            leaves["skip"] = s["skip"][i].detach().double().requires_grad_()
        if s["film"] is not None:
            leaves["film"] = s["film"][i].detach().double().requires_grad_()
        z = torch.cat([leaves["x"], leaves["skip"]], -1) if s["skip"] is not None else leaves["x"]
        z = z.reshape(per, case["groups"], -1)
        z = z - z.mean((0, 2), keepdim=True)
        z = z / ((z ** 2).mean((0, 2), keepdim=True) + 1e-5).sqrt()
        z = z.reshape(per, c) * wt + bs
        if s["film"] is not None:
            z = z + z * leaves["film"][:c] + leaves["film"][c:]
        if case["act"] == "silu":
            z = z / (1 + torch.exp(-z))
        if cut:
            z = z * ((_draws(i * per * c, per * c, s["rng"], "cuda") >= cut).double() * factor).reshape(per, c)
        z = z.reshape(case["h"], case["w"], c)
        rows["y"].append(z.detach())
        if train:
            gr = torch.autograd.grad(z, list(leaves.values()) + [wt, bs], s["dy"][i].double())
            for k, gk in zip(leaves, gr):
                rows["d" + k].append(gk)
            dwt += gr[-2]
            dbs += gr[-1]
    out = {"y": torch.stack(rows["y"])}
    if train:
        out.update({k: torch.stack(rows[k]) for k in ("dx", "dskip") if rows[k]}, dweight=dwt, dbias=dbs)
        if rows["dfilm"]:
            out["dfilm"] = torch.stack(rows["dfilm"])
    return out
