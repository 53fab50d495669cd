"""Cases and plain forms of the 8-bit activation checkpoints (``camal_amd.act_checkpoint``): what the training step keeps
of its forward pass for its backward pass, written, read back and used there.

Tensors are ``[window][time][channel]``.  A checkpoint holds the normalised values x = (z - mean) * invstd as 8-bit codes
with one power-of-two scale byte per 32 channels of a timestep.
"""
import math

import torch

own = False

BLOCK = 32
# format: (largest code value, added to the float's bits so that the exponent carries past it, exponent offset of the scale)
FORMATS = {"int8": (127.0, 0x1FFFF, 6), "e4m3": (448.0, 0x1FFFFF, 8)}


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the shortest training window of the narrowest model: latency
        dict(name="write short window", op="write", B=1, L=64, C=32, fmt="int8", skip=False),
        # the end of block 2 in a training batch of the default trainer: both branches are kept, their sum goes on
        dict(name="write batch with skip", op="write", B=128, L=510, C=128, fmt="int8", skip=True),
        # a batch of week windows at one-minute sampling
        dict(name="write week windows", op="write", B=24, L=10080, C=128, fmt="e4m3", skip=False),
        # a ragged last batch of odd windows, the activation of a block with its skip branch
        dict(name="read ragged batch", op="read", B=37, L=333, C=64, fmt="e4m3", skip=True),
        # a batch of day windows, widest model
        dict(name="read day windows", op="read", B=128, L=1440, C=256, fmt="int8", skip=False),
        # a handful of windows behind the temporal mean of the head: one gradient row per window
        dict(name="norm backward pooled", op="norm_backward", B=4, L=96, C=64, fmt="int8", relu=True, pooled=True),
        # the layer that a training step runs most often
        dict(name="norm backward batch", op="norm_backward", B=128, L=510, C=128, fmt="int8", relu=True, pooled=False),
        # week windows, widest model
        dict(name="norm backward weeks", op="norm_backward", B=24, L=10080, C=256, fmt="e4m3", relu=True, pooled=False),
        # the skip branch's 1x1 convolution, i.e. a linear layer
        dict(name="weight grad linear", op="weight_grad", B=128, L=510, cin=64, cout=128, ks=1, fmt="int8", skip=True, zero_pad=False),
        # the middle layer of blocks 2 and 3 in a training batch
        dict(name="weight grad 7 taps", op="weight_grad", B=128, L=510, cin=128, cout=128, ks=7, fmt="int8", skip=False, zero_pad=False),
        # the first layer of block 2 of the widest-kernel member, a ragged batch
        dict(name="weight grad 25 taps", op="weight_grad", B=37, L=333, cin=64, cout=128, ks=25, fmt="e4m3", skip=True, zero_pad=False),
        # the widest model on week windows, zeros outside the window
        dict(name="weight grad weeks", op="weight_grad", B=8, L=10080, cin=256, cout=256, ks=7, fmt="e4m3", skip=False, zero_pad=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "norm_backward", "weight_grad"])
    fmt = rng.choice(["int8", "e4m3"])
    L = _log_uniform(rng, 1, 10080)
    if op == "weight_grad":
        cin, cout = rng.choice([32, 64, 128, 256]), rng.choice([32, 64, 128, 256])
        ks = rng.choice([1, 3, 5, 7, 9, 15, 25])
        rows = min(80640, 80640 * 256 * 256 * 7 // (cin * cout * ks))
        return dict(op=op, B=_log_uniform(rng, 1, max(1, rows // L)), L=L, cin=cin, cout=cout, ks=ks, fmt=fmt,
                    skip=rng.random() < 0.4, zero_pad=rng.random() < 0.3)
    C = rng.choice([32, 64, 128, 256])
    case = dict(op=op, B=_log_uniform(rng, 1, max(1, 24 * 10080 * 128 // (C * L))), L=L, C=C, fmt=fmt)
    if op == "norm_backward":
        # over a handful of rows the normalisation leaves nothing of the gradient but its rounding: from 32 rows on
        case["B"] = max(case["B"], -(-32 // L))
        case.update(relu=rng.random() < 0.75, pooled=rng.random() < 0.25)
    else:
        case.update(skip=rng.random() < 0.4)
    return case


def work(case):
    B, L = case["B"], case["L"]
    if case["op"] == "weight_grad":
        cin, cout, ks = case["cin"], case["cout"], case["ks"]
        kept = (1 + 1 / BLOCK) * cin * (2 if case["skip"] else 1)
        return {"bytes": B * L * (4 * cout + kept) + 4 * cout * cin * ks, "flops": 2 * B * L * cout * cin * ks}
    n, kept = B * L * case["C"], 1 + 1 / BLOCK
    branches = 2 if case.get("skip") else 1
    if case["op"] == "write":  # z in, output and checkpoint out, the checkpoint read back as the values that it stands for
        return {"bytes": n * (4 * branches + 4 + branches * (2 * kept + 4)), "flops": 12 * n * branches}
    if case["op"] == "read":
        return {"bytes": n * (kept * branches + 4), "flops": 4 * n * branches}
    da = B * case["C"] if case["pooled"] else n
    return {"bytes": 4 * da + n * (kept + 4), "flops": 12 * n}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    """z of each branch with the statistics that go with it, and the layer's scale and shift."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    C = case.get("C") or case["cin"]
    B, L = case["B"], case["L"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def branch():
        # a quiet meter with bursts: most timesteps are small, some are several deviations out
        z = randn(B, L, C)
        z *= 0.4 + 2.0 * torch.rand(B, L, 1, device="cuda", generator=g) ** 8
        mean, std = 0.3 * randn(C), 0.5 + torch.rand(C, device="cuda", generator=g)
        z.mul_(std).add_(mean)
        var, mu = torch.var_mean(z.double(), dim=(0, 1), correction=0)
        invstd = (var + 1e-5).rsqrt().float()
        gamma = 1.0 + 0.25 * randn(C)
        gamma[::13] = -gamma[::13]
        return dict(z=z, mean=mu.float(), invstd=invstd, gamma=gamma, beta=0.3 * randn(C))

    main = branch()
    side = branch() if case.get("skip") else None
    return g, main, side


def prepare(case, seed):
    g, main, side = _inputs(case, seed)
    state = dict(case=dict(case), main=main, side=side)
    if case["op"] != "write":
        for b, relu in ((main, case.get("relu", True)), (side, False)):
            if b is not None:
                x = _normalised(b)
                k, exponent = _encode(x, b["gamma"], b["beta"], relu, case["fmt"])
                b["codes"], b["scales"] = _codes(k, case["fmt"]), exponent
                del b["z"]
    if case["op"] == "norm_backward":
        shape = (case["B"], case["C"]) if case["pooled"] else (case["B"], case["L"], case["C"])
        state["da"] = 1e-3 * torch.randn(*shape, device="cuda", generator=g)
    if case["op"] == "weight_grad":
        state["dz"] = 1e-3 * torch.randn(case["B"], case["L"], case["cout"], device="cuda", generator=g)
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _normalised(b):
    return (b["z"] - b["mean"]) * b["invstd"]


def _affine(x, gamma, beta):
    """gamma x + beta with one rounding: the ReLU's side must not depend on how many there were."""
    return torch.addcmul(beta.double(), x.double(), gamma.double()).float()


def _lattice(k, fmt):
    """What the k-th code from zero stands for, in units of the scale."""
    if fmt == "int8":
        return k.float()
    return _codes(k, fmt).float()


def _codes(k, fmt):
    if fmt == "int8":
        return k.to(torch.int8)
    return torch.where(k < 0, 128 - k, k).to(torch.uint8).view(torch.float8_e4m3fn)


def _encode(x, gamma, beta, relu, fmt):
    _, carry, offset = FORMATS[fmt]
    C = x.shape[-1]
    top = x.unflatten(-1, (C // BLOCK, BLOCK)).abs().amax(-1)
    exponent = (((top.view(torch.int32) + carry) >> 23) - offset).clamp_(min=1)
    scale = (exponent << 23).view(torch.float32).repeat_interleave(BLOCK, dim=-1)
    y = x / scale
    if fmt == "int8":
        k = y.round().to(torch.int32)
    else:
        byte = y.to(torch.float8_e4m3fn).view(torch.uint8).to(torch.int32)
        k = torch.where(byte >= 128, 128 - byte, byte)
    if relu:
        value = _lattice(k, fmt)
        wrong = (_affine(value * scale, gamma, beta) > 0) != (_affine(x, gamma, beta) > 0)
        k = torch.where(wrong, torch.where(value < y, k + 1, k - 1), k)
    return k, exponent.to(torch.uint8)


def _decode(b):
    scale = (b["scales"].to(torch.int32) << 23).view(torch.float32)
    return b["codes"].float() * scale.repeat_interleave(BLOCK, dim=-1)


def _activation(main, side):
    a = _affine(_decode(main), main["gamma"], main["beta"]).clamp_(min=0)
    return a if side is None else a + _affine(_decode(side), side["gamma"], side["beta"])


def _plain_write(case, main, side):
    x = _normalised(main)
    out = _affine(x, main["gamma"], main["beta"]).clamp_(min=0)
    k, exponent = _encode(x, main["gamma"], main["beta"], True, case["fmt"])
    kept = _decode(dict(codes=_codes(k, case["fmt"]), scales=exponent))
    if side is None:
        return {"out": out, "kept": kept}
    x = _normalised(side)
    out = out + _affine(x, side["gamma"], side["beta"])
    k, exponent = _encode(x, side["gamma"], side["beta"], False, case["fmt"])
    return {"out": out, "kept": kept, "kept_skip": _decode(dict(codes=_codes(k, case["fmt"]), scales=exponent))}


def _plain_norm_backward(case, b, da):
    n = case["B"] * case["L"]
    x = _decode(b)
    dy = (da / case["L"]).unsqueeze(1).expand_as(x) if case["pooled"] else da
    if case["relu"]:
        dy = dy * (_affine(x, b["gamma"], b["beta"]) > 0)
    dbeta = dy.sum((0, 1), dtype=torch.float64)
    dgamma = (dy * x).sum((0, 1), dtype=torch.float64)
    dz = b["gamma"] * b["invstd"] * (dy - (dbeta / n).float() - x * (dgamma / n).float())
    return {"dz": dz, "dgamma": dgamma.float(), "dbeta": dbeta.float()}


def _windowed(a, ks, zero_pad):
    """[B, L, C] -> [B, L + ks - 1, C]: the rows that the taps reach, edges repeated or zeros."""
    L = a.shape[1]
    at = torch.arange(-(ks // 2), L + ks // 2, device=a.device)
    rows = a.index_select(1, at.clamp(0, L - 1))
    return rows * ((at >= 0) & (at < L)).to(rows.dtype)[:, None] if zero_pad else rows


def _plain_weight_grad(case, main, side, dz):
    a = _activation(main, side).bfloat16().float()  # the operand of the product holds 8 significant bits
    taps = _windowed(a, case["ks"], case["zero_pad"]).unfold(1, case["ks"], 1)  # [B, L, cin, ks]
    dw = dz.reshape(-1, case["cout"]).t() @ taps.reshape(-1, case["cin"] * case["ks"])
    return dw.view(case["cout"], case["cin"], case["ks"])


def run(state):
    case, main, side = state["case"], state["main"], state["side"]
    if own:
        return _own(state, case, main, side)
    if case["op"] == "write":
        return _plain_write(case, main, side)
    if case["op"] == "read":
        return _activation(main, side)
    if case["op"] == "norm_backward":
        return _plain_norm_backward(case, main, state["da"])
    return _plain_weight_grad(case, main, side, state["dz"])


# ---- the framework's operators ----------------------------------------------------------------------------------------
def _own(state, case, main, side):
    from camal_amd import act_checkpoint as ac
    if case["op"] == "write":
        skip = side and (side["z"], side["mean"], side["invstd"], side["gamma"], side["beta"])
        got = ac.write(main["z"], main["mean"], main["invstd"], main["gamma"], main["beta"], fmt=case["fmt"], skip=skip)
        kept = {"out": got[0], "kept": ac.read(got[1])}
        return dict(kept, kept_skip=ac.read(got[2])) if side else kept
    ckpt = ac.ActivationCheckpoint(main["codes"], main["scales"])
    skip = side and (ac.ActivationCheckpoint(side["codes"], side["scales"]), side["gamma"], side["beta"])
    if case["op"] == "read":
        return ac.read(ckpt, main["gamma"], main["beta"], skip=skip)
    if case["op"] == "norm_backward":
        dz, dgamma, dbeta = ac.norm_backward(state["da"], ckpt, main["invstd"], main["gamma"], main["beta"], relu=case["relu"])
        return {"dz": dz, "dgamma": dgamma, "dbeta": dbeta}
    return ac.conv_weight_grad(state["dz"], ckpt, case["ks"], main["gamma"], main["beta"], skip=skip, zero_pad=case["zero_pad"])


# ---- in 64 bits, from the definitions ---------------------------------------------------------------------------------
def _power_of_two(k):
    return ((k.long() + 1023) << 52).view(torch.float64)  # torch.ldexp goes through pow, which need not be exact


def _exact_kept(x, gamma, beta, relu, fmt):
    """The checkpoint of the float32 values x (given in 64 bits): nearest point of the lattice, ties to even; with a ReLU
    the nearest of the two around x that lies on x's side of it."""
    largest = FORMATS[fmt][0]
    blocks = x.unflatten(-1, (-1, BLOCK))
    need = blocks.abs().amax(-1, keepdim=True) / largest
    mantissa, power = torch.frexp(need)
    power = torch.where(mantissa == 0.5, power - 1, power).clamp(min=-126)  # the smallest power of two >= need
    scale = _power_of_two(power).expand_as(blocks).flatten(-2)
    y = x / scale
    if fmt == "int8":
        step = torch.ones_like(y)
    else:  # three bits after the leading one, down to the fixed step of the subnormals
        step = _power_of_two((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    kept = (y / step).round() * step
    if relu:
        other = torch.where(kept < y, (y / step).ceil(), (y / step).floor()) * step
        bad = (gamma * (kept * scale) + beta > 0) != (gamma * x + beta > 0)
        kept = torch.where(bad, other, kept)
    return kept * scale


def _exact_values(b, relu, fmt):
    """x in 64 bits holding the float32 that the definition quantises: the difference and the product round once each."""
    x = ((b["z"].double() - b["mean"].double()).float().double() * b["invstd"].double()).float().double()
    return x, _exact_kept(x, b["gamma"].double(), b["beta"].double(), relu, fmt)


def exact(case, seed):
    g, main, side = _inputs(case, seed)
    x, kept = _exact_values(main, case.get("relu", True), case["fmt"])
    gamma, beta = main["gamma"].double(), main["beta"].double()
    if case["op"] == "norm_backward":
        n = case["B"] * case["L"]
        shape = (case["B"], case["C"]) if case["pooled"] else (case["B"], case["L"], case["C"])
        dy = (1e-3 * torch.randn(*shape, device="cuda", generator=g)).double()
        dy = (dy / case["L"])[:, None, :].expand(case["B"], case["L"], case["C"]) if case["pooled"] else dy
        if case["relu"]:
            dy = torch.where(gamma * kept + beta > 0, dy, 0.0)
        dbeta, dgamma = dy.sum((0, 1)), (dy * kept).sum((0, 1))
        return {"dz": gamma * main["invstd"].double() * (dy - dbeta / n - kept * (dgamma / n)), "dgamma": dgamma, "dbeta": dbeta}
    if side is not None:
        xs, kept_s = _exact_values(side, False, case["fmt"])
        gs, bs = side["gamma"].double(), side["beta"].double()
    if case["op"] == "write":
        out = torch.relu(gamma * x + beta)
        return {"out": out, "kept": kept} if side is None else {"out": out + gs * xs + bs, "kept": kept, "kept_skip": kept_s}
    a = torch.relu(gamma * kept + beta)
    if case["op"] == "read":
        return a if side is None else a + gs * kept_s + bs
    a = a.float()  # the operand is the float32 activation rounded to 8 significant bits
    a = (a if side is None else a + (gs * kept_s + bs).float()).bfloat16().double()
    dz = (1e-3 * torch.randn(case["B"], case["L"], case["cout"], device="cuda", generator=g)).double().reshape(-1, case["cout"])
    L, ks, at = case["L"], case["ks"], torch.arange(case["L"], device="cuda")
    dw = torch.empty(case["cout"], case["cin"], ks, dtype=torch.float64, device="cuda")
    for j in range(ks):
        p = at + j - ks // 2
        rows = a[:, p.clamp(0, L - 1)]
        if case["zero_pad"]:
            rows = rows * ((p >= 0) & (p < L)).double()[:, None]
        dw[:, :, j] = dz.t() @ rows.reshape(-1, case["cin"])
    return dw
