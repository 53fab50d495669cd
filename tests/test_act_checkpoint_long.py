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
