"""orthogonalise() / swg_orthogonalise and FusedMuonEMA against the formulas in float64 (tests/orth_ref.py, whose
emulation of the number formats gives the tolerances)."""
import ctypes as C

import pytest
import torch

from tests import orth_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _grad_mode():
    """Other modules of the suite switch gradients off for the process."""
    with torch.enable_grad():
        yield


def _gauss(shape, seed, t=F32):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(t)


def _spectrum(m, n, kind, seed):
    k = min(m, n)
    u, _ = torch.linalg.qr(_gauss((m, k), seed).double())
    v, _ = torch.linalg.qr(_gauss((n, k), seed + 1).double())
    s = {"decay": 10.0 ** (-4 * torch.arange(k) / k), "lowrank": torch.where(torch.arange(k) < max(1, k // 16), 1.0, 1e-5),
         "rank1": torch.where(torch.arange(k) < 1, 1.0, 0.0), "equal": torch.ones(k)}[kind].to(DEV).double()
    return ((u * s) @ v.t()).float()


def _check(g, out, steps=5, eps=1e-7):
    assert out.shape == g.shape and out.dtype in (BF16, F16)
    h = torch.finfo(out.dtype).eps / 2
    ref, each, norm = R.bounds(g, steps, eps)
    d = out.double() - ref
    assert float((d.abs() - h * (ref.abs() + each)).max()) <= each, (float(d.abs().max()), each)
    assert float(d.norm()) <= norm + h * float(ref.norm()), (float(d.norm()), norm)


# below, at and beyond the 32-wide padding, the 64- and 128-wide tiles, the transposed orientation of each
SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (1, 1000), (1000, 1), (31, 33), (32, 32), (33, 31), (33, 65), (60, 60), (60, 240), (64, 64),
          (65, 64), (96, 96), (96, 384), (384, 96), (120, 120), (129, 127), (127, 300), (192, 512), (251, 1003), (1003, 251),
          (257, 257), (40, 4099), (768, 512),
          # the one-workgroup form: each row class, its column classes and their ends, and just beyond them
          (20, 2048), (20, 2049), (32, 256), (300, 30), (32, 385), (64, 256), (64, 384), (64, 960), (1000, 60), (90, 600), (96, 640),
          (641, 96), (70, 386), (128, 256), (100, 257), (128, 384), (120, 360), (384, 121), (128, 385)]


@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape):
    import swingnn_amd as S
    g = _gauss(shape, shape[0] * 31 + shape[1])
    out = S.orthogonalise(g)
    _check(g, out)
    assert torch.equal(out, S.orthogonalise(g)), "equal inputs, equal bits"


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("out", [BF16, F16])
@pytest.mark.parametrize("shape", [(61, 200), (200, 61)])
def test_types(t, out, shape):
    import swingnn_amd as S
    g = _gauss(shape, 5, t)
    o = S.orthogonalise(g, out_dtype=out)
    assert o.dtype is out
    _check(g, o)


@pytest.mark.parametrize("kind", ["decay", "lowrank", "rank1", "equal"])
@pytest.mark.parametrize("shape", [(96, 384), (250, 250), (300, 70)])
def test_spectra(kind, shape):
    import swingnn_amd as S
    g = _spectrum(*shape, kind, 11)
    o = S.orthogonalise(g, out_dtype=F16)
    _check(g, o)
    if kind in ("rank1", "equal"):   # singular values of the result lie where the quintic sends them
        s = torch.linalg.svdvals(o.double())
        assert 0.6 < float(s[0]) < 1.25


@pytest.mark.parametrize("steps", [1, 2, 3, 6, 10])
def test_steps(steps):
    import swingnn_amd as S
    g = _gauss((70, 150), steps)
    _check(g, S.orthogonalise(g, steps=steps, out_dtype=F16), steps)


def test_large_tiles():
    """Enough 128-wide tiles that the wide form is taken (first assertion of the mixed list below keeps the narrow one)."""
    import swingnn_amd as S
    g = _gauss((48, 500, 530), 2)
    out = S.orthogonalise(g)
    for k in (0, 17, 47):
        _check(g[k], out[k])
    t = _gauss((48, 530, 500), 3)
    out = S.orthogonalise(t)
    for k in (0, 31, 47):
        _check(t[k], out[k])
    h = _gauss((1100, 3000), 4, BF16)
    _check(h, S.orthogonalise(h))


@pytest.mark.parametrize("shape", [(16, 4096), (130, 2500), (2048, 257), (65, 8192), (700, 2049), (2, 300, 2048), (1800, 4100),
                                   (4097, 1700)])
def test_long_contractions(shape):
    """A cut along the contraction: slices of uneven length, 64- and 128-wide tiles, batches, both orientations."""
    import swingnn_amd as S
    g = _gauss(shape, sum(shape))
    o = S.orthogonalise(g)
    for gg, oo in zip(g, o) if g.dim() == 3 else ((g, o),):
        _check(gg, oo)
    assert torch.equal(o, S.orthogonalise(g))
    pair = S.orthogonalise([g, _gauss((200, 40), 3)])    # beside a matrix with a short one
    _check(_gauss((200, 40), 3), pair[1])


def test_lists_of_mixed_shapes():
    import swingnn_amd as S
    shapes = [(3, 40, 96), (96, 96), (0, 5), (2, 300, 64), (64, 0), (0, 7, 7), (1, 1), (130, 260), (513, 33)]
    mats = [_gauss(s, i + 1) for i, s in enumerate(shapes)]
    outs = S.orthogonalise(mats)
    assert isinstance(outs, list) and [tuple(o.shape) for o in outs] == shapes
    for g, o in zip(mats, outs):
        if g.numel() == 0:
            continue
        for gg, oo in zip(g, o) if g.dim() == 3 else ((g, o),):
            _check(gg, oo)
    many = [_gauss((8 + k % 9, 5 + k % 7), k) for k in range(150)]   # more entries than one look at the table takes
    for g, o in zip(many, S.orthogonalise(many)):
        _check(g, o)
    assert S.orthogonalise([]) == [] and S.orthogonalise(torch.empty(0, 4, 4, device=DEV)).shape == (0, 4, 4)


def test_strides():
    import swingnn_amd as S
    wide = _gauss((6, 70, 150), 3)
    for g in (wide[1, :, 3:140], wide[:, :, :130], wide[::2, 1::3, 5:], wide[0].t(), wide.transpose(0, 1)[:, :, :9],
              wide[0, :1].expand(20, -1), wide[:, :, :1], wide[0, :, :1]):
        before = g.clone()
        o = S.orthogonalise(g)
        for gg, oo in zip(g, o) if g.dim() == 3 else ((g, o),):
            _check(gg, oo)
        assert torch.equal(g, before)


def test_scale_does_not_matter():
    import swingnn_amd as S
    g = _gauss((50, 90), 8)
    for f in (1e-28, 1e-12, 1e12, 1e30):
        _check(g * f, S.orthogonalise(g * f, eps=0.0), eps=0.0)
    _check(g * 1e-7, S.orthogonalise(g * 1e-7))          # eps counts here
    big = (g.half() * 1e4).clamp(-60000, 60000)
    _check(big, S.orthogonalise(big))


def test_zero_and_non_finite_matrices():
    import swingnn_amd as S
    g = _gauss((5, 40, 60), 9)
    g[1] = 0
    g[2, 3, 4] = float("nan")
    g[4, 39, 59] = float("inf")
    o = S.orthogonalise(g)
    assert not o[1].any() and bool(o[2].isnan().all()) and bool(o[4].isnan().all())
    for k in (0, 3):
        _check(g[k], o[k])


def test_non_finite_matrices_of_the_many_launch_form():
    import swingnn_amd as S
    g = _gauss((4, 150, 300), 9)
    g[1] = 0
    g[2, 149, 299] = float("inf")
    o = S.orthogonalise(g)
    assert not o[1].any() and bool(o[2].isnan().all())
    for k in (0, 3):
        _check(g[k], o[k])
    t = _gauss((2, 2300, 140), 5)               # a contraction in slices
    t[0, 7, 7] = float("nan")
    o = S.orthogonalise(t)
    assert bool(o[0].isnan().all())
    _check(t[1], o[1])


def test_small_ones_beside_a_long_one():
    import swingnn_amd as S
    mats = [_gauss((140, 2100), 1)] + [_gauss((30 + k, 50), k) for k in range(40)]
    for g, o in zip(mats, S.orthogonalise(mats)):
        _check(g, o)


def test_c_entry_leaves_gaps_alone_and_reads_its_strides():
    from swingnn_amd import _lib as L, engine as E
    g = _gauss((3, 50, 80), 4)
    for rows, cols in ((45, 71), (50, 13)):
        out = torch.full((3, 60, 90), 7.0, dtype=F16, device=DEV)
        it = (L.SwgOrthItem * 1)(L.SwgOrthItem(g.data_ptr(), out.data_ptr(), 80, 50 * 80, 90, 60 * 90, rows, cols, 3))
        nbytes = L.lib.swg_orthogonalise_workspace_bytes(1, it)
        ws = torch.full((nbytes,), 0xff, dtype=torch.uint8, device=DEV)   # NaN wherever something is read before it is written
        L.check(L.lib.swg_orthogonalise(1, it, 0, 2, 5, 1e-7, ws.data_ptr(), nbytes, E.stream_ptr()), "swg_orthogonalise")
        for k in range(3):
            _check(g[k, :rows, :cols], out[k, :rows, :cols])
        out[:, :rows, :cols] = 7.0
        assert bool((out == 7.0).all())


def test_streams_and_captured_graphs():
    """Two graphs captured one after the other, replayed in turn with new inputs and eager calls between."""
    import swingnn_amd as S
    a, b = _gauss((70, 90), 1), _gauss((2, 200, 64), 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = S.orthogonalise([a, b[0]])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], S.orthogonalise(a))
    graphs = []
    for t in (a, b):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = S.orthogonalise(t)
        graphs.append((gr, t, o))
    for seed in (5, 6, 7):
        for gr, t, o in graphs:
            t.copy_(_gauss(tuple(t.shape), seed))
            gr.replay()
            eager = S.orthogonalise(t)
            torch.cuda.synchronize()
            assert torch.equal(o, eager), seed


# ---- FusedMuonEMA ------------------------------------------------------------------------------------------------------
def _network(seed, big=False):
    """Parameters and how many of them are matrices; `big`: with matrices that only the many-launch form takes."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    shapes = [(96, 96), (288, 96), (96, 384), (17, 5), (1, 30), (61, 250), (250, 61)] + ([(200, 301), (513, 140)] if big else [])
    k = len(shapes)
    shapes += [(95,), (96,), (3, 4, 5), (1,), (2100,)]
    return [torch.nn.Parameter(0.05 * torch.randn(*s, device=DEV, generator=g)) for s in shapes], k


def _grads(params, seed, f=1e-2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    for p in params:
        p.grad = f * torch.randn(*p.shape, device=DEV, generator=g)


def _reference_step(st, k, grads, lr, mu, nesterov, wd, steps, max_norm, betas, eps, ema_decay):
    """One step in float64; -> bound of each parameter's error from the orthogonalised update."""
    clip = 1.0
    if max_norm is not None:
        norm = sum(float(g.double().square().sum()) for g in grads) ** 0.5
        clip = min(1.0, max_norm / (norm + 1e-6))
    st["t"] += 1
    tol = []
    for i, g in enumerate(grads):
        g = g.double() * clip
        p, m, v = st["p"][i], st["m"][i], st["v"][i]
        if i < k:
            m.mul_(mu).add_((1 - mu) * g)
            u = mu * m + (1 - mu) * g if nesterov else m
            o, each, _ = R.bounds(u, steps)
            f = lr * 0.2 * max(p.shape) ** 0.5
            p.mul_(1 - lr * wd).sub_(f * o)
            tol.append(f * each)
        else:
            g = g + wd * p
            m.mul_(betas[0]).add_((1 - betas[0]) * g)
            v.mul_(betas[1]).add_((1 - betas[1]) * g * g)
            p.sub_(lr * (m / (1 - betas[0] ** st["t"])) / ((v / (1 - betas[1] ** st["t"])).sqrt() + eps))
            tol.append(0.0)
        for j, d in enumerate(ema_decay):
            st["ema"][j][i].mul_(d).add_((1 - d) * p)
    return tol


@pytest.mark.parametrize("kw", [dict(), dict(nesterov=False, weight_decay=0.1), dict(max_norm=0.5, ema_betas=(0.9, 0.99)),
                                dict(ns_steps=3, momentum=0.0, ema_betas=(0.5,) * 8, weight_decay=0.01), dict(max_norm=1e9)])
@pytest.mark.parametrize("big", [False, True])
def test_optimizer_steps(kw, big):
    """Four steps against float64.  m, v: 4 roundings a step, 16 u in all of values that only grow; p: those of the update
    (the emulation's bound, added up over the steps) and 4 u |p| a step; Adam's quotient 16 u of its size lr / (1 - b1)."""
    import swingnn_amd as S
    params, k = _network(1, big)
    lr = 2e-3
    opt = S.FusedMuonEMA(params[:k], params[k:], lr=lr, **kw)
    st = {"t": 0, "p": [p.detach().double().clone() for p in params], "m": [torch.zeros_like(p, dtype=torch.float64) for p in params],
          "v": [torch.zeros_like(p, dtype=torch.float64) for p in params]}
    n_ema = len(kw.get("ema_betas", ()))
    st["ema"] = [[torch.zeros_like(p, dtype=torch.float64) for p in params] for _ in range(n_ema)]
    u, tol = 2.0 ** -24, [0.0] * len(params)
    for step in range(4):
        _grads(params, step)
        grads = [p.grad.clone() for p in params]
        decay = [0.0 if step < 2 else min(1 - 1 / (step + 1), b) for b in sorted(kw.get("ema_betas", ()))]
        version = [p._version for p in params]
        opt.step()
        more = _reference_step(st, k, grads, lr, kw.get("momentum", 0.95), kw.get("nesterov", True), kw.get("weight_decay", 0.0),
                               kw.get("ns_steps", 5), kw.get("max_norm"), (0.9, 0.999), 1e-8, decay)
        tol = [a + b for a, b in zip(tol, more)]
        assert all(p._version > v for p, v in zip(params, version))
        assert all(torch.equal(p.grad, g) for p, g in zip(params, grads)), "gradients stay as they are"
    if kw.get("max_norm") is not None:
        want = sum(float(g.double().square().sum()) for g in grads) ** 0.5
        assert abs(float(opt.grad_norm()) - want) <= 4 * u * want
    for i, p in enumerate(params):
        o = opt._offs[i]
        m, v = opt.m[o:o + p.numel()].view(p.shape).double(), opt.v[o:o + p.numel()].view(p.shape).double()
        gm = 1e-2 * 6
        assert float((m - st["m"][i]).abs().max()) <= 32 * u * gm, i
        adam = 0.0 if i < k else 4 * 64 * u * lr * 10
        bound = tol[i] + adam + 16 * u * (float(st["p"][i].abs().max()) + lr)
        assert float((p.detach().double() - st["p"][i]).abs().max()) <= bound, (i, bound)
        if i >= k:
            assert float((v - st["v"][i]).abs().max()) <= 32 * u * gm * gm
        for j in range(n_ema):
            e = opt.ema_parameters(j)[i].double()
            assert float((e - st["ema"][j][i]).abs().max()) <= bound + 16 * u, (i, j)


@pytest.mark.parametrize("big", [False, True])
def test_optimizer_repeats_itself_and_resumes(big):
    """Equal runs give equal bits; a run resumed from its checkpoint goes on as the uninterrupted one."""
    import swingnn_amd as S
    runs = []
    for resume in (False, False, True):
        params, k = _network(3, big)
        opt = S.FusedMuonEMA(params[:k], params[k:], lr=1e-3, max_norm=1.0, ema_betas=(0.9, 0.99))
        for step in range(5):
            if resume and step == 3:
                sd, old = opt.state_dict(), params
                params = [torch.nn.Parameter(p.detach().clone()) for p in old]
                opt = S.FusedMuonEMA(params[:k], params[k:], lr=7.0, max_norm=1.0, ema_betas=(0.9, 0.99))
                opt.load_state_dict(sd)
            _grads(params, step)
            opt.step()
        runs.append([p.detach().clone() for p in params] + [opt.m.clone(), opt.v.clone(), opt.ema.clone()])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_optimizer_without_others_and_moved_storage():
    import swingnn_amd as S
    p = torch.nn.Parameter(_gauss((40, 64), 1))
    opt = S.FusedMuonEMA([p], lr=1e-2)
    _grads([p], 1)
    opt.step()
    p.data = p.data.clone()
    p.grad = _gauss((64, 40), 5).t()           # not contiguous: taken as a copy
    before, g = p.detach().clone(), p.grad.clone()
    m = opt.m[:2560].view(40, 64).double()
    opt.step()
    want = before.double() - 1e-2 * 0.2 * 8 * R.exact(0.95 * (0.95 * m + 0.05 * g.double()) + 0.05 * g.double())
    assert float((p.detach().double() - want).abs().max()) < 1e-2 * 0.2 * 8 * 5e-3


@pytest.mark.parametrize("shapes", [[(33, 50), (7,)], [(160, 230), (300, 131), (9,)]])
def test_parameters_at_odd_addresses(shapes):
    """Views at 4-byte offsets, as slices of a flat buffer have them; what lies between them stays."""
    import swingnn_amd as S
    flat, gflat = torch.full((100000,), 3.0, device=DEV), _gauss((100000,), 1)
    at, params = 1, []
    for s in shapes:
        n = 1
        for d in s:
            n *= d
        flat[at:at + n] = 0.02 * _gauss((n,), n)
        params.append(torch.nn.Parameter(flat[at:at + n].view(s)))
        params[-1].grad = gflat[at + 2:at + 2 + n].view(s)
        at += n + 3
    before = flat.clone()
    opt = S.FusedMuonEMA(params[:-1], params[-1:], lr=1e-2, ema_betas=(0.9,))
    opt.step()
    torch.cuda.synchronize()
    at = 1
    for p in params:
        n = p.numel()
        if p.dim() == 2:
            ref, each, _ = R.bounds(0.05 * 1.95 * p.grad)
            f = 1e-2 * 0.2 * max(p.shape) ** 0.5
            want = before[at:at + n].view(p.shape).double() - f * ref
            assert float((p.detach().double() - want).abs().max()) <= f * each + 1e-7
        assert torch.equal(flat[at + n:at + n + 3], before[at + n:at + n + 3])
        at += n + 3
    assert torch.equal(flat[at:], before[at:])


def test_refused_checkpoints_and_groups():
    import swingnn_amd as S
    params, k = _network(5)
    opt = S.FusedMuonEMA(params[:k], params[k:], lr=1e-3)
    adam = S.FusedAdamEMA(params, lr=1e-3)
    with pytest.raises(ValueError):
        opt.load_state_dict(adam.state_dict())
    with pytest.raises(ValueError):
        adam.load_state_dict(opt.state_dict())
    with pytest.raises(ValueError):
        S.FusedMuonEMA(params[:k - 1], params[k - 1:], lr=1e-3).load_state_dict(opt.state_dict())
    with pytest.raises(NotImplementedError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, 2, device=DEV))]})
    with pytest.raises(NotImplementedError):
        opt.step(lambda: None)
    with pytest.raises(RuntimeError):
        opt.step()                              # no gradients
    _grads(params, 1)
    params[1].data = params[1].data.t().contiguous().t()
    with pytest.raises(NotImplementedError):
        opt.step()                              # rows and columns exchanged in memory
    params[1].data = params[1].data.contiguous()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
        with pytest.raises(NotImplementedError):
            opt.step()
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    opt.step()


@pytest.mark.parametrize("n_others", [0, 1, 700])
def test_gradient_norm(n_others):
    """grad_norm() against float64: one rounding to float32 of the sum and one of the root, and the same bits every time;
    more other parameters than workgroups that sum them."""
    import swingnn_amd as S
    mats = [torch.nn.Parameter(_gauss(s, i)) for i, s in enumerate([(96, 96), (3, 5), (300, 257)])]
    others = [torch.nn.Parameter(_gauss((1 + 37 * k,), k)) for k in range(n_others)]
    opt = S.FusedMuonEMA(mats, others, lr=0.0, max_norm=1.0)
    _grads(mats + others, 3, 1e3)
    want = sum(float(p.grad.double().square().sum()) for p in mats + others) ** 0.5
    got = []
    for _ in range(2):
        opt.step()
        got.append(float(opt.grad_norm()))
    assert got[0] == got[1] and abs(got[0] - want) <= 2.0 ** -23 * want


def test_update_that_cancels():
    """g = -a m / b: the update is nothing but rounding, its norm from the three sums is 1e-16 of the terms'."""
    import swingnn_amd as S
    p = torch.nn.Parameter(_gauss((64, 200), 1))
    opt = S.FusedMuonEMA([p], lr=1.0, momentum=0.5)
    opt.m.copy_(_gauss((64 * 200,), 2))
    p.grad = -(opt.m.view(64, 200) * (0.25 / 0.75))
    opt.step()
    assert bool(p.isfinite().all())


def test_training_run_together():
    """A small denoiser and a norm of the user's own, trained a few steps: the layer norm's gradients, the denoiser's, the
    split, the step.  Held: every parameter moves by what its rule allows, repeated runs agree bit for bit where the
    gradients do, and the weights the kernels derive follow (the loss of a second pass differs)."""
    import numpy as np
    import swingnn_amd as S
    torch.manual_seed(0)
    np.random.seed(0)
    net = S.SwinGNN(img_size=24, patch_size=3, in_chans=1, embed_dim=60, depths=[1, 1], num_heads=[3, 6], window_size=24,
                    mlp_ratio=4., drop_path_rate=0., self_condition=True)
    model = S.Precond("edm", net, True).to(DEV).train()
    norm = S.LayerNorm(24).to(DEV)
    both = torch.nn.ModuleList([model, norm])
    mats, others = S.FusedMuonEMA.split(both)
    assert len(mats) + len(others) == len(list(both.parameters())) and all(p.dim() == 2 for p in mats)
    assert not any(p.shape == net.down_layers[0].blocks[0].attn.relative_position_bias_table.shape for p in mats)
    opt = S.FusedMuonEMA(mats, others, lr=1e-3, max_norm=10.0, ema_betas=(0.9,))
    x = torch.randn(4, 24, 24, device=DEV)
    x, flags, sig = x + x.transpose(1, 2), torch.ones(4, 24, device=DEV), torch.full((4,), 0.5, device=DEV)
    losses = []
    for _ in range(3):
        opt.zero_grad(set_to_none=True)
        loss = (norm(model(x=x, node_flags=flags, sigmas=sig)) - x).square().mean()
        loss.backward()
        before = [p.detach().clone() for p in mats]
        opt.step()
        losses.append(float(loss.detach()))
        for p, q in zip(mats, before):
            moved = (p.detach() - q).square().mean().sqrt()
            # update_rms lr at most times 1.2024 (the largest singular value), sqrt(min / max) of it for a full matrix
            assert 0 < float(moved) <= 0.2 * 1e-3 * 1.25, tuple(p.shape)
        assert bool(norm.weight.grad.isfinite().all()) and bool((norm.weight.grad != 0).all())
    assert all(v == v for v in losses) and len(set(losses)) == 3
