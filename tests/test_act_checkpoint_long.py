"""8-bit activation checkpoints on calls long enough that every kernel goes round its loops, against 64-bit forms on the GPU."""
import pytest
import torch

gpu = pytest.mark.gpu
CHUNK = 1 << 17  # rows of a 64-bit product at once


def _tap(dz, a, ks, j, zero_pad=False):
    """sum_{b,t} dz[b][t][co] a[b][clamp(t + j - ks/2)][ci] in 64 bits."""
    L, cin = a.shape[1], a.shape[2]
    p = torch.arange(L, device=a.device) + j - ks // 2
    rows = a.index_select(1, p.clamp(0, L - 1))
    if zero_pad:
        rows = rows * ((p >= 0) & (p < L))[:, None]
    rows, d = rows.reshape(-1, cin), dz.reshape(-1, dz.shape[-1])
    out = torch.zeros(d.shape[1], cin, dtype=torch.float64, device=a.device)
    for k in range(0, d.shape[0], CHUNK):
        out += d[k:k + CHUNK].double().t() @ rows[k:k + CHUNK].double()
    return out


# ---- the weight gradient's chains of sums -------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("B,L,cin,cout,ks,taps", [(100, 10080, 256, 256, 63, (0, 31, 62)), (400, 10080, 256, 64, 15, (0, 14)),
                                                  (60000, 65, 128, 128, 3, (1,))])
def test_weight_grad_error_does_not_grow_with_the_rows(B, L, cin, cout, ks, taps):
    """dz and input of one sign, so that rounding has one, too.  A wave's chain is at most 8192 rows (4096 where windows are
    long): 3 products of 16 rows each, i.e. 1536 (768) sums, each cut off by at most 2^-23 of what it has reached, half of the
    last on average; then at most 16 + nsplit / 16 rounded sums of splits (nsplit < 1000) and 8 of waves."""
    from camal_amd import act_checkpoint as ac
    g = torch.Generator(device="cuda").manual_seed(1)
    one, zero = torch.ones(cin, device="cuda"), torch.zeros(cin, device="cuda")
    _, ckpt = ac.write(torch.randn(B, L, cin, device="cuda", generator=g), zero, one, one, zero)
    dz = torch.rand(B, L, cout, device="cuda", generator=g)
    dw = ac.conv_weight_grad(dz, ckpt, ks, one, zero)
    a = ac.read(ckpt, one, zero).bfloat16().float()
    sums = (1536 if 64 < L < 128 else 768) / 2
    for j in taps:
        want = _tap(dz, a, ks, j)
        assert ((dw[:, :, j].double() - want).abs() <= (sums * 2.0 ** -23 + 90 * 2.0 ** -24) * want).all(), j


# ---- every kernel on dense data past its first round ---------------------------------------------------------------------------
def _whole_numbers(B, L, ch, seed, fmt, top=4):
    """Normalised values that both formats hold exactly, and a scale and shift under which the activation is whole, too."""
    from camal_amd import act_checkpoint as ac
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-top, top + 1, (B, L, ch), device="cuda", generator=g).float()
    gamma = torch.randint(-2, 3, (ch,), device="cuda", generator=g).float()
    beta = torch.randint(-3, 4, (ch,), device="cuda", generator=g).float()
    zero, one = torch.zeros(ch, device="cuda"), torch.ones(ch, device="cuda")
    return x, gamma, beta, ac.write(x, zero, one, gamma, beta, relu=False, fmt=fmt)[1]


# Shapes of which a wave takes several units, for 1, 2 and 4 co tiles a workgroup and every size of tap group; last splits and last
# rounds that are not full; in the last three several sets of splits, the very last with a split that has no rows
@gpu
@pytest.mark.parametrize("fmt,skip,zero_pad", [("int8", False, False), ("e4m3", True, True)])
@pytest.mark.parametrize("B,L,cin,cout,ks", [
    (37, 333, 64, 128, 25), (128, 510, 64, 128, 1), (19, 517, 128, 128, 7), (3, 1111, 256, 256, 25), (2, 1300, 256, 256, 9),
    (101, 333, 128, 64, 7), (70, 650, 64, 64, 15), (30, 700, 256, 64, 3), (64, 700, 256, 32, 7), (90, 801, 128, 32, 25),
    (700, 70, 256, 32, 5), (9000, 17, 128, 128, 3), (5, 10079, 64, 256, 63), (1, 70001, 256, 128, 5), (300, 1440, 32, 32, 7), (100, 1440, 256, 256, 63),
    (30, 10079, 256, 128, 25), (8200, 333, 64, 64, 3)])
def test_weight_grad_of_whole_numbers(B, L, cin, cout, ks, fmt, skip, zero_pad):
    """Whole numbers whose sums stay below 2^24 in any order: nothing rounds, so the result is the exact one, bit for bit, or a
    row was lost, counted twice or taken from somewhere else.  |x| <= 4: |a| <= 2 4 + 3, twice that with the skip branch, and
    |dz| <= 8 of random sign; a sum of B L <= 2800000 such products stays below 8 22 sqrt(B L) 6 < 2^24 (six deviations of
    the largest; checked on the magnitudes that occur)."""
    from camal_amd import act_checkpoint as ac
    x, gamma, beta, ckpt = _whole_numbers(B, L, cin, 2, fmt)
    a = (x * gamma + beta).clamp(min=0)
    side = None
    if skip:
        xr, gr, br, ckpt_r = _whole_numbers(B, L, cin, 3, fmt)
        a += xr * gr + br
        side = (ckpt_r, gr, br)
    g = torch.Generator(device="cuda").manual_seed(4)
    dz = torch.randint(-8, 9, (B, L, cout), device="cuda", generator=g).float()
    assert torch.equal(ac.read(ckpt, gamma, beta, skip=side), a)
    dw = ac.conv_weight_grad(dz, ckpt, ks, gamma, beta, skip=side, zero_pad=zero_pad)
    for j in sorted({0, 1 % ks, ks // 2, ks - 1} | set(range(0, ks, 4))):
        want = _tap(dz, a, ks, j, zero_pad)
        assert want.abs().max() < 1 << 21
        assert torch.equal(dw[:, :, j].double(), want), j


@gpu
@pytest.mark.parametrize("B,L,cin,cout,ks", [(37, 333, 64, 128, 25), (128, 510, 128, 256, 7), (100, 333, 128, 64, 7), (90, 801, 128, 32, 5)])
def test_weight_grad_takes_all_of_dz(B, L, cin, cout, ks):
    """One step of each out-channel has a dz, with any 24 bits; the activation is 0 or a power of two.  Then every gradient is a
    single product of 24 bits, whose parts add up without rounding, and any piece of dz that got lost shows."""
    from camal_amd import act_checkpoint as ac
    g = torch.Generator(device="cuda").manual_seed(6)
    a = torch.tensor([0.0, 1.0, 2.0, 4.0], device="cuda")[torch.randint(0, 4, (B, L, cin), device="cuda", generator=g)]
    zero, one = torch.zeros(cin, device="cuda"), torch.ones(cin, device="cuda")
    _, ckpt = ac.write(a, zero, one, one, zero)
    co = torch.arange(cout, device="cuda")
    for rep in range(6):
        at = torch.randint(0, B * L, (cout,), device="cuda", generator=g)
        at[:4] = torch.tensor([0, L - 1, L, B * L - 1], device="cuda")
        v = torch.randint(-(1 << 24) + 1, 1 << 24, (cout,), device="cuda", generator=g).float() * 2.0 ** (10 * (rep - 3))
        dz = torch.zeros(B * L, cout, device="cuda")
        dz[at, co] = v
        dw = ac.conv_weight_grad(dz.view(B, L, cout), ckpt, ks, one, zero)
        b, t = at // L, at % L
        for j in range(ks):
            assert torch.equal(dw[:, :, j], v[:, None] * a[b, (t + j - ks // 2).clamp(0, L - 1)]), (rep, j)


LONG = [(67, 1023, 64), (33, 2001, 256), (200, 1003, 32), (131, 1009, 256), (1, 70001, 128), (40000, 3, 128)]


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("B,L,ch", LONG)
def test_norm_backward_of_whole_numbers(B, L, ch, fmt):
    """|x| <= 4, |da| <= 8 (a multiple of L where all steps share it): both sums are whole numbers that nothing rounds (fp32
    sums over a lane's rows stay below 2^24), so they are exact or a row was lost or counted twice.  dz rounds: the means once
    each, then gamma invstd, two differences and three products."""
    from camal_amd import act_checkpoint as ac
    x, gamma, beta, ckpt = _whole_numbers(B, L, ch, 7, fmt)
    invstd = 0.5 + torch.rand(ch, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(8)
    n = B * L
    for relu in (True, False):
        for pooled in (False, True):
            da = torch.randint(-8, 9, (B, ch) if pooled else (B, L, ch), device="cuda", generator=g).float()
            dy = (da[:, None, :].expand(B, L, ch) if pooled else da).double()
            if relu:
                dy = torch.where(x * gamma + beta > 0, dy, 0.0)
            dz, dgamma, dbeta = ac.norm_backward(da * L if pooled else da, ckpt, invstd, gamma, beta, relu=relu)
            s1, s2 = dy.sum((0, 1)), (dy * x).sum((0, 1))
            assert s1.abs().max() < 1 << 24 and s2.abs().max() < 1 << 24
            assert torch.equal(dbeta.double(), s1) and torch.equal(dgamma.double(), s2)
            gi = gamma.double() * invstd.double()
            want = gi * (dy - s1 / n - x * (s2 / n))
            terms = dy.abs() + (s1 / n).abs() + (x * (s2 / n)).abs()
            assert ((dz.double() - want).abs() <= 7 * 2.0 ** -24 * gi.abs() * terms).all()


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("B,L,ch", [(67, 1023, 64), (33, 2001, 256), (1, 140001, 128)])
def test_write_and_read_many_rows(B, L, ch, fmt):
    """Codes and scales of every element, both branches, against the 64-bit form."""
    from camal_amd import act_checkpoint as ac
    from tests import act_reference as ref
    g = torch.Generator(device="cuda").manual_seed(9)

    def branch():
        z = torch.randn(B, L, ch, device="cuda", generator=g) * torch.rand(B, L, 1, device="cuda", generator=g) ** 4
        v = [torch.randn(ch, device="cuda", generator=g) for _ in range(4)]
        return z, 0.1 * v[0], 1 + 0.2 * v[1].abs(), 1 + 0.3 * v[2], 0.3 * v[3]

    main, side = branch(), branch()
    out, ckpt, ckpt_r = ac.write(*main, fmt=fmt, skip=side)
    x, xr = ref.normalised(*main[:3]), ref.normalised(*side[:3])
    kept, e = ref.keep(x, fmt, *main[3:])
    kept_r, e_r = ref.keep(xr, fmt)
    assert torch.equal(ckpt.scales, e) and torch.equal(ckpt_r.scales, e_r)
    assert torch.equal(ac.read(ckpt).double(), kept) and torch.equal(ac.read(ckpt_r).double(), kept_r)
    back = ac.read(ckpt, *main[3:], skip=(ckpt_r, *side[3:]))
    for got, v, vr in ((out, x, xr), (back, kept, kept_r)):
        want = ref.activation(v, *main[3:], skip=(vr, *side[3:]))
        u, ur = ref.affine(v, *main[3:]).abs(), ref.affine(vr, *side[3:]).abs()
        assert ((got.double() - want).abs() <= 2.0 ** -24 * (u + ur + want.abs()) * 1.01).all()
