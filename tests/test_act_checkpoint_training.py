"""Training steps with 8-bit activation checkpoints: the forward pass is the fp32 step's bit for bit, the checkpoints are what
their definition says, and every gradient is that of a 64-bit backward pass on the values that they hold."""
import ctypes as C

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from camal_amd import weights
from tests import act_reference as ref

gpu = pytest.mark.gpu


def _model(k, arch, mid, seed=31):
    from camal_amd.resnet import CamALResNet, ResNet
    torch.manual_seed(seed)
    m = ResNet(mid_channels=mid) if arch == "resnet" else CamALResNet(kernel_size=k, mid_channels=mid)
    g = np.random.default_rng(seed)
    for key in m._params:  # scales of both signs, shifts that put thresholds into the data
        if m._params[key].ndim == 1 and key.endswith((".weight", ".bias")) and m._params[key].size > 2:
            v = 0.3 * g.standard_normal(m._params[key].size).astype(np.float32)
            m._params[key] = v + (np.where(g.random(v.size) < 0.15, -1, 1).astype(np.float32) if key.endswith(".weight") else 0)
    return m


def _layers(eng):
    """The flat parameter vector cut up as include/camal_hip.h lays it out: per layer (conv.w, conv.b, gamma, beta), then the head."""
    c1, c2 = eng.mid, 2 * eng.mid
    ks = (7, 5, 3) if eng.arch == weights.ARCH_RESNET else (eng.k, 7, 3)
    shapes = [(1, c1, ks[0]), (c1, c1, ks[1]), (c1, c1, ks[2]), (1, c1, 1), (c1, c2, ks[0]), (c2, c2, ks[1]), (c2, c2, ks[2]),
              (c1, c2, 1), (c2, c2, ks[0]), (c2, c2, ks[1]), (c2, c2, ks[2])]

    def cut(flat):
        out, o = [], 0
        for cin, cout, k in shapes:
            sizes = [cout * cin * k, cout, cout, cout]
            parts = [flat[o + sum(sizes[:i]):o + sum(sizes[:i + 1])] for i in range(4)]
            out.append([parts[0].view(cout, cin, k), *parts[1:]])
            o += sum(sizes)
        return out, flat[o:o + 2 * c2].view(2, c2), flat[o + 2 * c2:]
    return cut


def _data_grad(dz, w, L, zero_pad):
    """Gradient of the convolution's input [B, L, Cin] in 64 bits."""
    a = torch.zeros(dz.shape[0], w.shape[1], L, dtype=torch.float64, requires_grad=True)
    p = w.shape[2] // 2
    padded = F.pad(a, (p, p)) if zero_pad or p == 0 else F.pad(a, (p, p), mode="replicate")
    out = F.conv1d(padded, w.double())
    return torch.autograd.grad(out, a, dz.transpose(1, 2))[0].transpose(1, 2)


def _backward64(eng, x, y, feat, kept, invstd, params):
    """Every gradient, from the kept values in 64 bits.  Slots 0..10 in the order of the parameters."""
    layers, wfc, bfc = _layers(eng)(params)
    zpad, B, L = eng.arch == weights.ARCH_RESNET, *x.shape
    grads = [[None] * 4 for _ in layers]
    pooled = feat.double().mean(1)
    p = torch.softmax(pooled @ wfc.double().t() + bfc.double(), 1)
    dl = (p - F.one_hot(y.long(), 2)) / B
    head = (dl.t() @ pooled, dl.sum(0))
    da = dl @ wfc.double()

    def norm(slot, da, relu):
        w = layers[slot]
        dz, grads[slot][2], grads[slot][3], _ = ref.norm_backward(da, kept[slot], invstd[slot], w[2], w[3], relu)
        return dz

    def wgrad(slot, dz, src):
        if src is None:
            a = x.double()[..., None]
        else:
            s, skip = src
            a = ref.operand(kept[s], layers[s][2], layers[s][3], skip=None if skip is None else (kept[skip], layers[skip][2], layers[skip][3]))
        grads[slot][0] = ref.weight_grad(dz, a, layers[slot][0].shape[2], zpad)[0]

    # (slot, its input as (slot, skip slot))
    blocks = [[(0, None), (1, (0, None)), (2, (1, None))], [(4, (2, 3)), (5, (4, None)), (6, (5, None))],
              [(8, (6, 7)), (9, (8, None)), (10, (9, None))]]
    skips = [(3, None), (7, (2, 3)), None]
    for b in (2, 1, 0):
        side = None
        if skips[b]:
            slot, src = skips[b]
            side = norm(slot, da, False)
            wgrad(slot, side, src)
        for slot, src in reversed(blocks[b]):
            dz = norm(slot, da, True)
            wgrad(slot, dz, src)
            if src is not None:
                da = _data_grad(dz, layers[slot][0], L, zpad)
        if b == 1:
            da = da + _data_grad(side, layers[7][0], L, zpad)
    return grads, head


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("k,B,L,arch,mid", [(7, 5, 64, "camal", 64), (25, 3, 97, "camal", 64), (5, 4, 33, "camal", 32),
                                            (9, 2, 70, "camal", 128), (7, 3, 81, "resnet", 64), (3, 37, 5, "camal", 64),
                                            (15, 1, 200, "camal", 32), (63, 2, 40, "camal", 64), (7, 1, 1, "camal", 64)])
def test_step_against_a_64_bit_backward_on_the_checkpoints(k, B, L, arch, mid, fmt):
    from camal_amd import synth
    from camal_amd.trainer import TrainEngine
    m = _model(k, arch, mid)
    x, y = synth.ideal_windows(B, L, seed=5)
    x, y = torch.as_tensor(x).float(), torch.as_tensor(y).int()
    full = TrainEngine(m, "cuda:0", B + 2, L + 3)
    eng = TrainEngine(m, "cuda:0", B + 2, L + 3, act_checkpoint=fmt)
    assert 0 < eng.workspace_bytes < full.workspace_bytes
    loss0, nc0 = (t.clone() for t in full.forward_backward(x, y))
    loss1, nc1 = (t.clone() for t in eng.forward_backward(x, y))
    # the forward pass is the same one
    assert torch.equal(loss0, loss1) and torch.equal(nc0, nc1) and torch.equal(full.running, eng.running)
    params = eng.params.cpu()
    layers, _, _ = _layers(eng)(params)
    kept, invstd = [], []
    for slot in range(11):
        mean, istd = full.peek("mean", slot, B, L).cpu(), full.peek("invstd", slot, B, L).cpu()
        assert torch.equal(istd, eng.peek("invstd", slot, B, L).cpu())
        xs = ref.normalised(full.peek("z", slot, B, L).cpu(), mean, istd)
        want, _ = ref.keep(xs, fmt, *((layers[slot][2], layers[slot][3]) if slot not in (3, 7) else ()))
        assert torch.equal(eng.peek("xhat", slot, B, L).cpu().double(), want), slot
        kept.append(want)
        invstd.append(istd)
    feat = full.peek("act", 8, B, L).cpu()
    grads, head = _backward64(eng, x, y, feat, kept, invstd, params)
    got, hw, hb = _layers(eng)(eng.grads.cpu().double())
    # 22 passes from the loss to the first layer, each a chain of fp32 sums of at most 256 * 63 products (norm-wise
    # error at most sqrt(16128) 2^-24 = 8e-6, the step's own float32 kernels among them): 2e-4, as 1e-3 of the largest gradient
    top = max(float(t.abs().max()) for g in grads for t in g if t is not None)
    for slot in range(11):
        for i in (0, 2, 3):
            err = (got[slot][i] - grads[slot][i]).abs().max()
            assert err <= 1e-3 * max(float(grads[slot][i].abs().max()), 1e-2 * top), (slot, i, float(err))
        assert (got[slot][1] == 0).all()  # a bias in front of a BatchNorm
    assert (hw - head[0]).abs().max() <= 1e-4 * head[0].abs().max() and (hb - head[1]).abs().max() <= 1e-4
    full.close()
    eng.close()


@gpu
def test_ragged_batches_and_two_call_criterion():
    """Smaller batches on a larger workspace give what a workspace of their size gives, bit for bit; a caller's criterion
    (forward, its gradient, backward) agrees with the built-in cross-entropy."""
    from camal_amd import synth
    from camal_amd.trainer import TrainEngine
    m = _model(9, "camal", 64)
    big = TrainEngine(m, "cuda:0", 16, 90, act_checkpoint="int8")
    for B, L in ((16, 90), (3, 41), (1, 90), (16, 7)):
        x, y = synth.ideal_windows(B, L, seed=B)
        own = TrainEngine(m, "cuda:0", B, L, act_checkpoint="int8")
        big.forward_backward(x, y)
        own.forward_backward(x, y)
        assert torch.equal(big.grads, own.grads), (B, L)
        ce = big.grads.clone()
        big.forward_backward(x, y, criterion=torch.nn.CrossEntropyLoss())
        # the two softmaxes differ by a few roundings; every gradient is linear in their result
        assert (big.grads - ce).abs().max() <= 1e-4 * ce.abs().max()
        own.close()
    big.close()


@gpu
def test_steps_on_streams_and_in_a_graph():
    """Members side by side on streams of their own, and a step captured into a graph, give the eager step's gradients."""
    from camal_amd import synth
    from camal_amd.trainer import MemberStreams, TrainEngine
    x, y = synth.ideal_windows(6, 70, seed=2)
    xd, yd = torch.as_tensor(x).float().cuda(), torch.as_tensor(y).to(torch.int32).cuda()
    models = [_model(k, "camal", 64, seed=k) for k in (5, 7, 25)]
    alone = []
    for mdl, fmt in zip(models, ("int8", "e4m3", "int8")):
        e = TrainEngine(mdl, "cuda:0", 6, 70, data_parallel=False, act_checkpoint=fmt)
        for _ in range(3):
            e.forward_backward(xd, yd)
            e.optimizer_step(1e-3, 0.0)
        alone.append(e.params.clone())
        e.close()
    engines = [TrainEngine(mdl, "cuda:0", 6, 70, data_parallel=False, act_checkpoint=fmt)
               for mdl, fmt in zip(models, ("int8", "e4m3", "int8"))]
    side = MemberStreams(engines)
    for _ in range(3):
        side.step(xd, yd, 1e-3, 0.0)
    torch.cuda.synchronize()
    assert all(torch.equal(e.params, a) for e, a in zip(engines, alone))
    e = engines[0]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        e.forward_backward(xd, yd, update_running=False)
    other = TrainEngine(models[0], "cuda:0", 6, 70, data_parallel=False, act_checkpoint="int8")
    for rep in range(4):
        xd.mul_(0.9).add_(0.01 * rep)
        e.params.mul_(1.001)
        g.replay()
        other.params.copy_(e.params)
        other.forward_backward(xd, yd, update_running=False)
        torch.cuda.synchronize()
        assert torch.equal(other.grads, e.grads) and torch.equal(other.loss, e.loss), rep
    for e in (*engines, other):
        e.close()


@gpu
def test_trainer_and_camal_take_the_option():
    from camal_amd import CamAL, synth
    from camal_amd.resnet import CamALResNet
    from camal_amd.trainer import BasedClassifTrainer, TSLoader
    x, y = synth.ideal_windows(48, 64, seed=3)
    tr = BasedClassifTrainer(CamALResNet(kernel_size=7), TSLoader(x, y, batch_size=20), device="cuda:0", act_checkpoint="e4m3")
    tr.train(2)
    assert tr.engine.act_checkpoint == "e4m3" and np.isfinite(tr.loss_train_history).all()
    camal = CamAL(n_predictors=1, device="cuda:0")
    camal.train((x[:32], y[:32]), (x[32:40], y[32:40]), (x[40:], y[40:]), list_kernel_sizes=[5], epochs=2, batch_size=16, act_checkpoint="int8")
    assert camal.camal_logs["is_fitted"] and camal.predict(x[40:]).shape == (8, 64)


@gpu
def test_peek_and_create_refusals():
    from camal_amd import _lib
    from camal_amd.trainer import TrainEngine
    m = _model(5, "camal", 32)
    with pytest.raises(ValueError):
        TrainEngine(m, "cuda:0", 2, 16, act_checkpoint="int4")
    full, eng = TrainEngine(m, "cuda:0", 2, 16), TrainEngine(m, "cuda:0", 2, 16, act_checkpoint="int8")
    x = torch.randn(2, 16)
    full.forward_train(x)
    eng.forward_train(x)
    for e, what in ((full, "xhat"), (eng, "z"), (eng, "act")):
        with pytest.raises(_lib.CamalHipError):
            e.peek(what, 0, 2, 16)
    with pytest.raises(_lib.CamalHipError):
        eng.peek("xhat", 11, 2, 16)
    h = C.c_void_p()
    lib = _lib.load()
    assert lib.camal_trainer_create_act(0, 5, 2, 16, 0, 32, 2, C.byref(h)) == -1
    assert lib.camal_trainer_create_act(0, 5, 1 << 16, 1 << 16, 0, 32, 0, C.byref(h)) == -1
    assert lib.camal_trainer_workspace_bytes(None) == 0
    full.close()
    eng.close()


@gpu
@pytest.mark.parametrize("fmt,mid,B,L", [(None, 64, 5, 70), ("int8", 64, 5, 70), ("e4m3", 32, 3, 41), ("int8", 128, 2, 130)])
def test_one_forward_pass_serves_several_backward_passes(fmt, mid, B, L):
    """Gradients of several losses of one batch: each is what a forward pass of its own gives, bit for bit, whatever ran
    backward before it."""
    from camal_amd import _lib, synth
    from camal_amd.trainer import TrainEngine
    eng = TrainEngine(_model(7, "camal", mid), "cuda:0", B, L, act_checkpoint=fmt)
    x, y = synth.ideal_windows(B, L, seed=9)
    x, y = torch.as_tensor(x).float().cuda().contiguous(), torch.as_tensor(y).int().cuda().contiguous()
    g = torch.Generator().manual_seed(1)
    losses = [torch.randn(B, 2, generator=g).cuda() / B for _ in range(3)]

    def backward(dlogits):
        _lib.check(eng.lib.camal_train_bwd_dlogits(eng._h, _lib.ptr(eng.params), _lib.ptr(x), _lib.ptr(y), _lib.ptr(dlogits), B, L,
                                                   _lib.ptr(eng.grads), _lib.ptr(eng.loss), _lib.ptr(eng.ncorrect), eng._stream()))
        return eng.grads.clone(), eng.loss.clone()

    own = []
    for d in losses:
        eng.forward_train(x)
        own.append(backward(d))
    eng.forward_train(x)
    for _ in range(2):
        for d, want in zip(losses, own):
            got = backward(d)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    eng.forward_backward(x, y, update_running=False)  # a whole step is a forward pass, too
    assert torch.equal(backward(losses[0])[0], own[0][0])
    eng.close()


@gpu
@pytest.mark.parametrize("k,mid", [(25, 32), (7, 64)])
def test_long_batches_on_a_longer_workspace(k, mid):
    """Batches of over a million timesteps, whose weight gradients are summed in several sets: a shorter batch on the workspace
    of a longer one gives what it gives on its own, bit for bit."""
    from camal_amd import synth
    from camal_amd.trainer import TrainEngine
    if torch.cuda.mem_get_info()[0] < 32 << 30:
        pytest.skip("needs 32 GB of GPU memory")
    m = _model(k, "camal", mid)
    big = TrainEngine(m, "cuda:0", 230, 10080, act_checkpoint="int8")
    for B, L in ((230, 10080), (113, 10080), (229, 9970)):
        g = torch.Generator(device="cuda").manual_seed(B)
        x = torch.randn(B, L, device="cuda", generator=g)
        y = (torch.arange(B, device="cuda") % 2).to(torch.int32)
        own = TrainEngine(m, "cuda:0", B, L, act_checkpoint="int8")
        big.forward_backward(x, y)
        own.forward_backward(x, y)
        assert torch.isfinite(own.grads).all() and own.grads.abs().max() > 0
        assert torch.equal(big.grads, own.grads), (B, L)
        own.close()
    big.close()
