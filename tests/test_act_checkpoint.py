"""8-bit activation checkpoints against plain 64-bit forms on the CPU: codes and scales exactly, sums within the bounds of
fp32 arithmetic, at the sizes, values and masks where they can go wrong; refusals; streams, strides, graphs."""
import ctypes as C

import pytest
import torch

from tests import act_reference as ref

U = 2.0 ** -24  # unit roundoff of float32
FMTS = ["int8", "e4m3"]
gpu = pytest.mark.gpu


def _norm(ch, seed, z):
    g = torch.Generator().manual_seed(seed)
    flat = z.double().reshape(-1, ch)
    mean = flat.mean(0).float()
    invstd = (flat.var(0, unbiased=False) + 1e-5).rsqrt().float()
    gamma = 1.0 + 0.3 * torch.randn(ch, generator=g)
    gamma[::5] *= -1
    gamma[7::16] = 0.0
    beta = 0.3 * torch.randn(ch, generator=g)
    beta[3::11] = 0.0
    return mean, invstd, gamma, beta


def _z(B, L, ch, seed):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(B, L, ch, generator=g) * torch.rand(B, L, 1, generator=g) ** 4
    return z * (0.2 + torch.rand(ch, generator=g)) + torch.randn(ch, generator=g)


def _dev(*t):
    return [x.cuda() if torch.is_tensor(x) else x for x in t]


def _values(ckpt):
    s = torch.pow(2.0, ckpt.scales.cpu().double() - 127).repeat_interleave(ref.BLOCK, dim=-1)
    return ckpt.codes.cpu().float().double() * s


SHAPES = [(1, 1, 32), (1, 1, 256), (2, 1, 64), (1, 2, 128), (3, 7, 32), (5, 13, 64), (1, 129, 128), (4, 257, 32), (7, 61, 256)]


# ---- the definition itself, on the CPU -----------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FMTS)
def test_reference_keeps_the_mask_and_stays_within_a_step(fmt):
    """What the format promises, checked on the plain form: every mask bit survives, no element moves by a step or more,
    and rounding alone (the plain form without gamma) would have flipped some."""
    z = _z(6, 200, 64, 3)
    mean, invstd, gamma, beta = _norm(64, 4, z)
    x = ref.normalised(z, mean, invstd)
    kept, e = ref.keep(x, fmt, gamma, beta)
    near, _ = ref.keep(x, fmt)
    side = ref.affine(x, gamma, beta) > 0
    assert torch.equal(ref.affine(kept, gamma, beta) > 0, side)
    assert (ref.affine(near, gamma, beta) > 0).ne(side).float().mean() > 1e-3
    s = torch.pow(2.0, e.double() - 127).repeat_interleave(32, -1)
    step = s if fmt == "int8" else s * torch.pow(2.0, torch.floor(torch.log2((x / s).abs().clamp(min=2.0 ** -6))) - 3)
    assert ((kept - x).abs() < step).all() and ((near - x).abs() <= step / 2).all()
    assert (kept.abs() <= ref.LARGEST[fmt] * s).all()


def test_python_refusals():
    from camal_amd import _lib
    from camal_amd import act_checkpoint as ac
    z, v = torch.zeros(2, 3, 64), torch.ones(64)
    with pytest.raises(_lib.CamalHipError):
        ac.write(z, v, v, v, v)  # no CPU path
    with pytest.raises(ValueError):
        ac.write(torch.zeros(2, 3, 48), v, v, v, v)
    with pytest.raises(ValueError):
        ac.write(z, v, v, v, v, fmt="int4")
    codes, scales = torch.zeros(2, 3, 64, dtype=torch.int8), torch.ones(2, 3, 2, dtype=torch.uint8)
    ckpt = ac.ActivationCheckpoint(codes, scales)
    assert ckpt.fmt == "int8" and ckpt.nbytes == 2 * 3 * 66 and tuple(ckpt.shape) == (2, 3, 64)
    for c, s in ((codes.float(), scales), (codes, scales.int()), (codes, scales[..., :1]), (codes[0], scales[0]),
                 (torch.zeros(2, 3, 96, dtype=torch.int8), torch.ones(2, 3, 3, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            ac.ActivationCheckpoint(c, s)
    for call in (lambda: ac.read(ckpt), lambda: ac.norm_backward(z, ckpt, v, v, v), lambda: ac.conv_weight_grad(z, ckpt, 3, v, v)):
        with pytest.raises(_lib.CamalHipError):
            call()


def test_c_entry_refusals():
    """Every refusal happens on the host, before anything is launched (this test runs where there is no GPU)."""
    from camal_amd import _lib
    lib = _lib.load()
    P = C.c_void_p(1 << 20)  # never dereferenced
    odd = C.c_void_p((1 << 20) + 4)

    def write(z=P, out=P, codes=P, rows=5, ch=64, fmt=0, zr=None, codes_r=None):
        return lib.camal_act_write(z, P, P, P, P, 1, zr, P, P, P, P, rows, ch, fmt, out, codes, P, codes_r, P, None)

    bad = [write(z=None), write(out=None), write(codes=None), write(rows=0), write(rows=-1), write(rows=1 << 31), write(ch=48),
           write(ch=512), write(fmt=2), write(z=odd), write(codes=C.c_void_p((1 << 20) + 2)), write(zr=P), write(zr=odd, codes_r=P)]

    def read(codes=P, g=P, b=P, relu=1, codes_r=None, g_r=P, out=P, rows=5, ch=64, fmt=0):
        return lib.camal_act_read(codes, P, fmt, rows, ch, g, b, relu, codes_r, P, g_r, P, out, None)

    bad += [read(codes=None), read(g=None), read(b=None), read(g=None, b=None), read(g=None, b=None, relu=0, codes_r=P),
            read(codes_r=P, g_r=None), read(out=odd), read(rows=0), read(ch=31), read(fmt=-1)]

    def bwd(da=P, B=2, L=3, ch=64, fmt=0, ws=P, nbytes=1 << 30, dg=P):
        return lib.camal_act_norm_bwd(da, 0, P, P, fmt, B, L, ch, P, P, P, 1, P, dg, P, ws, nbytes, None)

    need = lib.camal_act_norm_bwd_workspace_bytes(6, 64)
    bad += [bwd(da=None), bwd(B=0), bwd(L=0), bwd(B=1 << 16, L=1 << 15), bwd(ch=33), bwd(fmt=7), bwd(ws=None), bwd(nbytes=need - 1),
            bwd(dg=None), bwd(da=odd)]

    def wgrad(dz=P, B=2, L=3, cin=64, cout=64, ks=3, fmt=0, codes_r=None, g_r=P, ws=P, nbytes=1 << 40, dw=P):
        return lib.camal_act_wgrad(dz, P, P, fmt, B, L, cin, cout, ks, P, P, 1, codes_r, P, g_r, P, 0, dw, ws, nbytes, None)

    need_w = lib.camal_act_wgrad_workspace_bytes(2, 3, 64, 64, 3)
    bad += [wgrad(dz=None), wgrad(B=0), wgrad(L=0), wgrad(B=1 << 16, L=1 << 15), wgrad(cin=48), wgrad(cout=16), wgrad(ks=2), wgrad(ks=0),
            wgrad(ks=65), wgrad(fmt=3), wgrad(codes_r=P, g_r=None), wgrad(ws=None), wgrad(nbytes=need_w - 1), wgrad(dw=None), wgrad(dz=odd)]
    assert bad == [-1] * len(bad)
    assert lib.camal_act_norm_bwd_workspace_bytes(0, 64) == 0 == lib.camal_act_norm_bwd_workspace_bytes(5, 40)
    assert lib.camal_act_wgrad_workspace_bytes(2, 3, 64, 64, 4) == 0 and need > 0 and need_w >= 4 * 64 * 64 * 3


# ---- write and read --------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("B,L,ch", SHAPES)
def test_write_and_read_back(B, L, ch, fmt):
    from camal_amd import act_checkpoint as ac
    z, zr = _z(B, L, ch, 1), _z(B, L, ch, 2)
    n, nr = _norm(ch, 3, z), _norm(ch, 4, zr)
    x, xr = ref.normalised(z, *n[:2]), ref.normalised(zr, *nr[:2])
    for relu in (True, False):
        for skip in (False, True):
            got = ac.write(*_dev(z, *n), relu=relu, fmt=fmt, skip=_dev(zr, *nr) if skip else None)
            kept, e = ref.keep(x, fmt, *(n[2:] if relu else ()))
            assert got[1].fmt == fmt and torch.equal(got[1].scales.cpu(), e) and torch.equal(_values(got[1]), kept)
            assert torch.equal(ac.read(got[1]).cpu().double(), kept)
            u, ur = ref.affine(x, *n[2:]), ref.affine(xr, *nr[2:])
            want = ref.activation(x, *n[2:], relu=relu, skip=(xr, *nr[2:]) if skip else None)
            # u rounds once, and with a skip branch so do u_r and the sum
            tol = U * (u.abs() + (ur.abs() + want.abs() if skip else 0)) * 1.01
            assert ((got[0].cpu().double() - want).abs() <= tol).all()
            back = ac.read(got[1], *_dev(*n[2:]), relu=relu, skip=(got[2], *_dev(*nr[2:])) if skip else None).cpu().double()
            kept_r, e_r = ref.keep(xr, fmt)
            if skip:
                assert torch.equal(got[2].scales.cpu(), e_r) and torch.equal(_values(got[2]), kept_r)
            uk, ukr = ref.affine(kept, *n[2:]), ref.affine(kept_r, *nr[2:])
            want = ref.activation(kept, *n[2:], relu=relu, skip=(kept_r, *nr[2:]) if skip else None)
            assert ((back - want).abs() <= U * (uk.abs() + (ukr.abs() + want.abs() if skip else 0)) * 1.01).all()
            if relu:
                assert torch.equal(uk > 0, u > 0)


@gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_write_special_values(fmt):
    """Ties, scale borders, zero blocks, tiny and huge values, infinities and NaNs, zero and negative gamma: mean 0 and
    invstd 1, so x = z."""
    from camal_amd import act_checkpoint as ac
    big = ref.LARGEST[fmt]
    z = torch.zeros(12, 1, 64)
    z[0, 0, :32] = torch.arange(32) + 0.5                      # ties under a scale of 1
    z[0, 0, 31] = big
    z[1, 0, :32] = -(torch.arange(32) + 0.5)
    z[1, 0, 31] = -big
    z[2, 0, 0] = big * (1 + 2.0 ** -23)                         # one bit past what the scale holds
    z[2, 0, 1] = -big
    z[3, 0, :4] = torch.tensor([1e-38, -3e-39, 1e-45, 5e-42])   # down to subnormals
    z[4, 0, :4] = torch.tensor([3.4e38, -1e38, 1.0, -1e-30])
    z[5, 0, :3] = torch.tensor([float("inf"), 1.0, -2.0])
    z[6, 0, 5] = float("nan")
    z[7, 0, 5] = -float("inf")
    z[7, 0, 32:] = torch.linspace(-2, 2, 32)                    # the block beside it is not touched
    z[8] = -0.0
    z[9, 0] = torch.tensor([2.0 ** -k for k in range(64)])
    z[10, 0] = -torch.tensor([1.0 + 2.0 ** -(k + 1) for k in range(64)])
    z[11, 0] = torch.linspace(-1e-3, 1e-3, 64)
    g = torch.Generator().manual_seed(0)
    for gamma in (torch.ones(64), -torch.ones(64), torch.zeros(64), 1e-20 * torch.ones(64), torch.randn(64, generator=g)):
        for beta in (torch.zeros(64), 0.25 * torch.ones(64), -1e-4 * torch.ones(64), -0.75 * torch.ones(64)):
            n = (torch.zeros(64), torch.ones(64), gamma, beta)
            out, ckpt = ac.write(*_dev(z, *n), fmt=fmt)
            x = z.double()
            kept, e = ref.keep(x, fmt, gamma, beta)
            assert torch.equal(ckpt.scales.cpu(), e)
            back = ac.read(ckpt).cpu().double()
            off = torch.nonzero((back != kept) & ~(back.isnan() & kept.isnan()))
            assert off.numel() == 0, [(tuple(i.tolist()), x[tuple(i)].item(), back[tuple(i)].item(), kept[tuple(i)].item()) for i in off[:5]]
            fine = torch.isfinite(kept)
            want = ref.activation(x, gamma, beta)
            assert torch.equal(out.cpu().isnan(), want.isnan())
            assert torch.equal(ref.side(back, gamma, beta)[fine], ref.side(x, gamma, beta)[fine])


# ---- norm backward -----------------------------------------------------------------------------------------------------------
def _bwd_tolerance(m, x):
    """fp32 chains of at most 64 terms, then 64-bit sums: (64 + 3) U of the magnitudes (the mask is exact; the pooled
    gradient's division rounds once).  dz: both means enter with their error, the rest rounds at most five times."""
    t1, t2 = 67 * U * m["abs1"], 67 * U * m["abs2"]
    n = m["n"]
    terms = m["dy"].abs() + (m["abs1"] / n) + x.abs() * (m["abs2"] / n)
    return t1, t2, m["gi"] * (t1 / n + x.abs() * t2 / n + 6 * U * terms)


@gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("B,L,ch", SHAPES + [(2, 64, 64), (1, 65, 256), (66, 1, 32), (3, 1000, 64)])
def test_norm_backward(B, L, ch, fmt):
    from camal_amd import act_checkpoint as ac
    z = _z(B, L, ch, 5)
    n = _norm(ch, 6, z)
    x = ref.normalised(z, *n[:2])
    g = torch.Generator().manual_seed(7)
    for relu in (True, False):
        kept, _ = ref.keep(x, fmt, *(n[2:] if relu else ()))
        _, ckpt = ac.write(*_dev(z, *n), relu=relu, fmt=fmt)
        for da in (torch.randn(B, L, ch, generator=g), torch.randn(B, ch, generator=g)):
            dz, dgamma, dbeta = ac.norm_backward(da.cuda(), ckpt, *_dev(*n[1:]), relu=relu)
            wz, wg, wb, m = ref.norm_backward(da, kept, *n[1:], relu=relu)
            t1, t2, tz = _bwd_tolerance(m, kept)
            assert ((dbeta.cpu().double() - wb).abs() <= t1 + 1e-30).all()
            assert ((dgamma.cpu().double() - wg).abs() <= t2 + 1e-30).all()
            assert ((dz.cpu().double() - wz).abs() <= tz + 1e-30).all()


@gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_norm_backward_against_differences(fmt):
    """Values that the formats hold exactly, with mean 0 and mean square 1, so that the checkpoint changes nothing: the
    gradient against central differences of the whole BatchNorm + ReLU in 64 bits."""
    from camal_amd import act_checkpoint as ac
    g = torch.Generator().manual_seed(8)
    col = torch.tensor([2.5, 1, .5, .5, .5, 0, 0, 0])
    col = torch.cat([col, -col])
    x = torch.stack([col[torch.randperm(16, generator=g)] for _ in range(32)], 1).reshape(2, 8, 32)
    std, mean = 0.25 + torch.rand(32, generator=g), torch.zeros(32)
    std = torch.pow(2.0, torch.floor(torch.log2(std)))
    gamma, beta = 1 + 0.3 * torch.randn(32, generator=g), 0.2 + 0.1 * torch.rand(32, generator=g)
    z, up = x * std, torch.randn(2, 8, 32, generator=g)
    out, ckpt = ac.write(*_dev(z, mean, 1 / std, gamma, beta), fmt=fmt)
    assert torch.equal(_values(ckpt), x.double())
    dz, dgamma, dbeta = (t.cpu().double() for t in ac.norm_backward(up.cuda(), ckpt, *_dev(1 / std, gamma, beta)))

    def loss(zz, gg, bb):
        m, v = zz.mean((0, 1)), zz.var((0, 1), unbiased=False)
        return (torch.relu(gg * (zz - m) / v.sqrt() + bb) * up.double()).sum()

    z64, g64, b64 = z.double(), gamma.double(), beta.double()
    h = 1e-5  # differences are off by h^2 times third derivatives (about 1e-9) and by rounding over h (about 1e-10)

    def differences(args, k):
        d = torch.zeros_like(args[k])
        for i in range(d.numel()):
            e = torch.zeros_like(d).view(-1)
            e[i] = h
            hi, lo = list(args), list(args)
            hi[k], lo[k] = args[k] + e.view_as(d), args[k] - e.view_as(d)
            d.view(-1)[i] = (loss(*hi) - loss(*lo)) / (2 * h)
        return d

    args = [z64, g64, b64]
    for k, got in enumerate((dz, dgamma, dbeta)):
        want = differences(args, k)
        assert ((got - want).abs() <= 1e-5 * want.abs().max()).all()


# ---- weight gradient -----------------------------------------------------------------------------------------------------------
def _wgrad_case(B, L, cin, cout, ks, fmt, relu=True, skip=False, zero_pad=False, seed=11):
    from camal_amd import act_checkpoint as ac
    z, zr = _z(B, L, cin, seed), _z(B, L, cin, seed + 1)
    n, nr = _norm(cin, seed + 2, z), _norm(cin, seed + 3, zr)
    got = ac.write(*_dev(z, *n), relu=relu, fmt=fmt, skip=_dev(zr, *nr) if skip else None)
    dz = torch.randn(B, L, cout, generator=torch.Generator().manual_seed(seed + 4))
    dw = ac.conv_weight_grad(dz.cuda(), got[1], ks, *_dev(*n[2:]), relu=relu, skip=(got[2], *_dev(*nr[2:])) if skip else None,
                             zero_pad=zero_pad)
    kept, _ = ref.keep(ref.normalised(z, *n[:2]), fmt, *(n[2:] if relu else ()))
    kept_r, _ = ref.keep(ref.normalised(zr, *nr[:2]), fmt)
    a = ref.operand(kept, *n[2:], relu=relu, skip=(kept_r, *nr[2:]) if skip else None)
    want, mag = ref.weight_grad(dz, a, ks, zero_pad)
    # exact operands, at most three products for each of the B L terms, summed in fp32 in some order
    assert dw.shape == want.shape
    assert ((dw.cpu().double() - want).abs() <= (3 * B * L + 8) * U * mag * 1.01 + 1e-30).all()


@gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("B,L,cin,cout,ks", [
    (1, 1, 32, 32, 1), (1, 1, 32, 32, 7), (9, 1, 64, 32, 3), (1, 2, 32, 64, 5), (5, 3, 64, 64, 15), (2, 15, 128, 32, 3),
    (2, 16, 32, 128, 7), (2, 17, 64, 128, 1), (1, 31, 128, 128, 9), (3, 32, 256, 32, 3), (1, 33, 32, 256, 5), (2, 63, 64, 64, 7),
    (2, 64, 128, 128, 7), (2, 65, 64, 128, 25), (1, 127, 256, 256, 3), (1, 128, 128, 256, 1), (3, 129, 32, 32, 63), (1, 300, 64, 64, 9),
    (40, 5, 128, 64, 7), (3, 200, 256, 64, 15)])
def test_weight_grad(B, L, cin, cout, ks, fmt):
    _wgrad_case(B, L, cin, cout, ks, fmt)
    _wgrad_case(B, L, cin, cout, ks, fmt, skip=True, zero_pad=True)


@gpu
@pytest.mark.parametrize("relu,skip,zero_pad", [(False, False, False), (False, True, False), (True, True, False), (True, False, True)])
def test_weight_grad_forms(relu, skip, zero_pad):
    _wgrad_case(3, 70, 64, 128, 7, "int8", relu, skip, zero_pad)
    _wgrad_case(2, 90, 32, 64, 3, "e4m3", relu, skip, zero_pad)


@gpu
@pytest.mark.parametrize("cin", [32, 64, 128, 256])
@pytest.mark.parametrize("cout", [32, 64, 128, 256])
def test_weight_grad_every_channel_pair(cin, cout):
    for ks in (1, 3, 5, 7):
        _wgrad_case(2, 50, cin, cout, ks, "int8")


@gpu
@pytest.mark.parametrize("ks", list(range(1, 64, 2)))
def test_weight_grad_every_kernel_size(ks):
    _wgrad_case(2, 40, 32, 64, ks, "e4m3")


@gpu
def test_weight_grad_wide_range_of_dz():
    """dz over 40 binary orders of magnitude, and a value that rounds past the largest bf16: all 24 bits take part."""
    from camal_amd import act_checkpoint as ac
    g = torch.Generator().manual_seed(3)
    z = _z(1, 96, 32, 9)
    n = _norm(32, 10, z)
    _, ckpt = ac.write(*_dev(z, *n))
    kept, _ = ref.keep(ref.normalised(z, *n[:2]), "int8", *n[2:])
    a = ref.operand(kept, *n[2:])
    dz = torch.randn(1, 96, 32, generator=g) * torch.pow(2.0, -40 * torch.rand(1, 1, 32, generator=g))
    dz[0, :, 0] *= 2.0 ** -60
    want, mag = ref.weight_grad(dz, a, 3)
    dw = ac.conv_weight_grad(dz.cuda(), ckpt, 3, *_dev(*n[2:])).cpu().double()
    assert ((dw - want).abs() <= (3 * 96 + 8) * U * mag * 1.01).all()
    one = torch.zeros(1, 96, 32)
    one[0, 10, 4] = torch.finfo(torch.float32).max / 64
    one[0, 20, 5] = 1 + 2.0 ** -23
    want, mag = ref.weight_grad(one, a, 1)
    dw = ac.conv_weight_grad(one.cuda(), ckpt, 1, *_dev(*n[2:])).cpu().double()
    assert ((dw - want).abs() <= 4 * U * mag).all()


@gpu
def test_nan_reaches_what_depends_on_it():
    from camal_amd import act_checkpoint as ac
    z = _z(2, 40, 64, 12)
    n = _norm(64, 13, z)
    z[1, 20, 40] = float("nan")
    _, ckpt = ac.write(*_dev(z, *n))
    assert ac.read(ckpt)[1, 20, 32:].isnan().all() and not ac.read(ckpt)[..., :32].isnan().any()
    da = torch.randn(2, 40, 64)
    dz, dgamma, _ = ac.norm_backward(da.cuda(), ckpt, *_dev(*n[1:]))
    assert dgamma[32:].isnan().all() and not dgamma[:32].isnan().any()
    assert dz[..., 32:].isnan().all() and not dz[..., :32].isnan().any()
    dw = ac.conv_weight_grad(da.cuda(), ckpt, 3, *_dev(*n[2:]))
    assert dw[:, 32:].isnan().all() and not dw[:, :32].isnan().any()


# ---- how they are called -------------------------------------------------------------------------------------------------------
def _run_all(ac, z, zr, n, nr, da, dz, ks=5, fmt="int8"):
    out, ckpt, side = ac.write(z, *n, fmt=fmt, skip=(zr, *nr))
    got = [out, ckpt.codes.view(torch.uint8), ckpt.scales, side.codes.view(torch.uint8), side.scales,
           ac.read(ckpt, *n[2:], skip=(side, *nr[2:]))]
    got += ac.norm_backward(da, ckpt, *n[1:])
    got.append(ac.conv_weight_grad(dz, ckpt, ks, *n[2:], skip=(side, *nr[2:])))
    return got


def _inputs(B=3, L=77, ch=64, cout=128, seed=20):
    z, zr = _z(B, L, ch, seed), _z(B, L, ch, seed + 1)
    n, nr = _norm(ch, seed + 2, z), _norm(ch, seed + 3, zr)
    g = torch.Generator().manual_seed(seed + 4)
    return _dev(z, zr), _dev(*n), _dev(*nr), torch.randn(B, L, ch, generator=g).cuda(), torch.randn(B, L, cout, generator=g).cuda()


@gpu
def test_strides_offsets_and_streams():
    """Transposed, sliced and misaligned inputs, and a stream of the caller's, give what dense ones give, bit for bit."""
    from camal_amd import act_checkpoint as ac
    (z, zr), n, nr, da, dz = _inputs()
    want = _run_all(ac, z, zr, n, nr, da, dz)

    def other(t):
        flat = torch.empty(t.numel() + 1, device="cuda")[1:]  # 4 bytes past an aligned address
        flat.copy_(t.reshape(-1))
        return flat.view(t.shape)

    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (z, zr, da, dz)]
    got = _run_all(ac, turned[0], turned[1], n, nr, turned[2], turned[3])
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = _run_all(ac, other(z), other(zr), [other(t) for t in n], [other(t) for t in nr], other(da), other(dz))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run_all(ac, z, zr, n, nr, da, dz)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@gpu
def test_two_streams_at_once():
    """Calls that overlap on two streams have workspaces of their own: the same results as one after the other."""
    from camal_amd import act_checkpoint as ac
    sets = [_inputs(B=16, L=300, seed=60), _inputs(B=9, L=510, ch=128, cout=64, seed=70)]
    want = [_run_all(ac, *i[0], *i[1:]) for i in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, (st, i) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[k].append(_run_all(ac, *i[0], *i[1:]))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(a, b) for r in runs for a, b in zip(w, r))


@gpu
def test_sliced_and_turned_checkpoints():
    """A slice of a checkpoint (its scales start at any byte) and one whose memory is laid out otherwise."""
    from camal_amd import act_checkpoint as ac
    (z, _), n, _, da, dz = _inputs(B=5, L=33, ch=32)
    _, ckpt = ac.write(z, *n, fmt="e4m3")
    _, few = ac.write(z[1:4], *n, fmt="e4m3")
    want = [ac.read(few), *ac.norm_backward(da[1:4], few, *n[1:]), ac.conv_weight_grad(dz[1:4], few, 3, *n[2:])]
    turn = lambda t: t.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(t.dtype)  # noqa: E731
    for c in (ac.ActivationCheckpoint(ckpt.codes[1:4], ckpt.scales[1:4]),
              ac.ActivationCheckpoint(turn(few.codes), turn(few.scales))):
        got = [ac.read(c), *ac.norm_backward(da[1:4], c, *n[1:]), ac.conv_weight_grad(dz[1:4], c, 3, *n[2:])]
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@gpu
def test_captured_and_replayed():
    """Two graphs of the whole run, replayed in turns with new inputs and eager work in between."""
    from camal_amd import act_checkpoint as ac
    sets = [_inputs(seed=30), _inputs(B=2, L=130, seed=40)]
    graphs = []
    for (z, zr), n, nr, da, dz in sets:
        _run_all(ac, z, zr, n, nr, da, dz)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = _run_all(ac, z, zr, n, nr, da, dz)
        graphs.append((g, outs))
    for rep in range(4):
        for (g, outs), ((z, zr), n, nr, da, dz) in zip(graphs, sets):
            z.mul_(1.0 + 0.1 * rep).add_(0.01)
            da.neg_()
            g.replay()
            want = _run_all(ac, z, zr, n, nr, da, dz)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), rep


@gpu
def test_offsets_beyond_32_bits():
    """2.2e9 elements: the last rows come out as in a call of their own."""
    from camal_amd import act_checkpoint as ac
    rows, ch, tail = 8_600_000, 256, 70
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of GPU memory")
    g = torch.Generator(device="cuda").manual_seed(1)
    z = torch.zeros(1, rows, ch, device="cuda")
    z[:, -tail:] = torch.randn(1, tail, ch, device="cuda", generator=g)
    n = _dev(torch.zeros(ch), torch.ones(ch), *_norm(ch, 5, torch.zeros(1, 4, ch))[2:])
    out, ckpt = ac.write(z, *n, fmt="e4m3")
    few, own = ac.write(z[:, -tail:], *n, fmt="e4m3")
    assert torch.equal(out[:, -tail:], few) and torch.equal(ckpt.scales[:, -tail:], own.scales)
    assert torch.equal(ckpt.codes[:, -tail:].view(torch.uint8), own.codes.view(torch.uint8))
    assert torch.equal(ac.read(ckpt)[:, -tail:], ac.read(own))
    del out
    z.zero_()
    z[:, -tail:] = torch.randn(1, tail, ch, device="cuda", generator=g)  # now the gradient: all in the last rows
    dz, dgamma, dbeta = ac.norm_backward(z, ckpt, *n[1:])
    kept = _values(own)
    wz, wg, wb, m = ref.norm_backward(z[:, -tail:].cpu(), kept, *(t.cpu() for t in n[1:]))
    t1, t2, _ = _bwd_tolerance(m, kept)
    assert ((dbeta.cpu().double() - wb).abs() <= t1).all() and ((dgamma.cpu().double() - wg).abs() <= t2).all()
    side = (n[2] * n[1] * torch.where(ac.read(own) * n[2] + n[3] > 0, z[:, -tail:], 0.0))
    assert (dz[:, -tail:] - side).abs().max() <= 1e-4 * side.abs().max()  # the means are 1e-7 of it: 1.2e5 times fewer rows
    del dz
    dw = ac.conv_weight_grad(z, ckpt, 3, *n[2:])
    a = ref.operand(kept, *(t.cpu() for t in n[2:]))
    base = ref.operand(torch.zeros(1, 1, ch, dtype=torch.float64), *(t.cpu() for t in n[2:]))
    want, mag = ref.weight_grad(torch.cat([torch.zeros(1, 1, ch), z[:, -tail:].cpu()], 1), torch.cat([base, a], 1), 3)
    assert ((dw.cpu().double() - want).abs() <= (3 * tail + 8) * U * mag * 1.01).all()


@gpu
def test_rows_behind_the_last_stay_as_they_were():
    """The C entry points write exactly rows * channels elements."""
    from camal_amd import _lib
    lib = _lib.load()
    rows, ch, cout, ks = 37, 64, 32, 3
    z = _z(1, rows, ch, 50)
    n = _dev(*_norm(ch, 51, z))
    z = z.cuda()
    out = torch.full((rows + 9, ch), 7.0, device="cuda")
    codes, scales = torch.full((rows + 9, ch), 99, dtype=torch.uint8, device="cuda"), torch.full((rows + 9, ch // 32), 99, dtype=torch.uint8, device="cuda")
    _lib.check(lib.camal_act_write(_lib.ptr(z), *map(_lib.ptr, n), 1, None, None, None, None, None, rows, ch, 0, _lib.ptr(out),
                                   _lib.ptr(codes), _lib.ptr(scales), None, None, None))
    back, dz = torch.full((rows + 9, ch), 7.0, device="cuda"), torch.full((rows + 9, ch), 7.0, device="cuda")
    _lib.check(lib.camal_act_read(_lib.ptr(codes), _lib.ptr(scales), 0, rows, ch, None, None, 0, None, None, None, None, _lib.ptr(back), None))
    sums = torch.full((2, 3, ch), 7.0, device="cuda")
    need = lib.camal_act_norm_bwd_workspace_bytes(rows, ch)
    ws = torch.full((need + 64,), 77, dtype=torch.uint8, device="cuda")
    _lib.check(lib.camal_act_norm_bwd(_lib.ptr(z), 0, _lib.ptr(codes), _lib.ptr(scales), 0, 1, rows, ch, *map(_lib.ptr, n[1:]), 1,
                                      _lib.ptr(dz), _lib.ptr(sums[0, 1]), _lib.ptr(sums[1, 1]), _lib.ptr(ws), need, None))
    dw = torch.full((3, cout, ch, ks), 7.0, device="cuda")
    need_w = lib.camal_act_wgrad_workspace_bytes(1, rows, ch, cout, ks)
    ws_w = torch.full((need_w + 64,), 77, dtype=torch.uint8, device="cuda")
    d = torch.randn(rows, cout, device="cuda")
    _lib.check(lib.camal_act_wgrad(_lib.ptr(d), _lib.ptr(codes), _lib.ptr(scales), 0, 1, rows, ch, cout, ks, *map(_lib.ptr, n[2:]), 1,
                                   None, None, None, None, 0, _lib.ptr(dw[1]), _lib.ptr(ws_w), need_w, None))
    torch.cuda.synchronize()
    for t, v in ((out, 7.0), (codes, 99), (scales, 99), (back, 7.0), (dz, 7.0)):
        assert (t[rows:] == v).all() and not (t[:rows] == v).all()
    assert (sums[:, 0] == 7).all() and (sums[:, 2] == 7).all() and (sums[:, 1] != 7).all()
    assert (dw[0] == 7).all() and (dw[2] == 7).all() and (dw[1] != 7).any()
    assert (ws[need:] == 77).all() and (ws_w[need_w:] == 77).all()


@gpu
def test_device_refusals():
    from camal_amd import act_checkpoint as ac
    (z, zr), n, nr, da, dz = _inputs(1, 5, 64, 32)
    _, ckpt = ac.write(z, *n)
    _, other = ac.write(z, *n, fmt="e4m3")
    calls = [lambda: ac.write(z.half(), *n), lambda: ac.write(z, n[0][:32], *n[1:]), lambda: ac.write(z, *n, skip=(zr[:, :4], *nr)),
             lambda: ac.write(z, *n, skip=(zr, *nr[:3])), lambda: ac.write(z, n[0].cpu(), *n[1:]), lambda: ac.read(ckpt, n[2]),
             lambda: ac.read(ckpt, skip=(other, n[2], n[3])), lambda: ac.read(ckpt, *n[2:], skip=(other, *n[2:])),
             lambda: ac.norm_backward(da[:, :3], ckpt, *n[1:]), lambda: ac.norm_backward(da.double(), ckpt, *n[1:]),
             lambda: ac.conv_weight_grad(dz[..., :16], ckpt, 3, *n[2:]), lambda: ac.conv_weight_grad(dz[:, :3], ckpt, 3, *n[2:])]
    for call in calls:
        with pytest.raises(ValueError):
            call()
    from camal_amd import _lib
    for ks in (0, 2, 65, -1):
        with pytest.raises(_lib.CamalHipError):
            ac.conv_weight_grad(dz, ckpt, ks, *n[2:])
    with pytest.raises(_lib.CamalHipError):
        ac.write(z[:, :0], *n)


@gpu
def test_kernel_size_is_a_whole_number():
    from camal_amd import _lib
    from camal_amd import act_checkpoint as ac
    (z, _), n, _, _, dz = _inputs(1, 9, 64, 32)
    _, ckpt = ac.write(z, *n)
    for ks in (3.5, 1.25, 7.999):
        with pytest.raises(_lib.CamalHipError):
            ac.conv_weight_grad(dz, ckpt, ks, *n[2:])
    assert torch.equal(ac.conv_weight_grad(dz, ckpt, 3.0, *n[2:]), ac.conv_weight_grad(dz, ckpt, 3, *n[2:]))
