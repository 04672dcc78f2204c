"""grad_norm, clip_grad_norm_ and FusedSGD.step(max_norm=...) on the GPU against double precision.

Tolerances.  u = torch.finfo(dtype).eps / 2.  The norm: squares and sums in double (relative error below 1e-9 at these sizes), rounded
to fp32 once: 2^-24 |norm|.  A clipped gradient: the factor is rounded to fp32 (2^-24), the product to fp32 (2^-24) and to the
gradient's type (u), or half the type's smallest step."""
import math

import pytest
import torch

from yolov6_amd.solver import FusedSGD, LossScaler, clip_grad_norm_, grad_norm
from yolov6_amd.train_engine import ParamArena

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _norm64(grads, p):
    every = torch.cat([g.double().reshape(-1) for g in grads])
    return float(every.abs().max() if p == math.inf else every.abs().sum() if p == 1 else every.square().sum().sqrt())


def _params(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty_like(g))
        p.grad = g
        out.append(p)
    return out


def _check_clip(grads, max_norm, p=2.0):
    before = [g.clone() for g in grads]
    norm = clip_grad_norm_(_params(grads), max_norm, p)
    want = _norm64(before, p)
    assert norm.dtype == torch.float32 and norm.shape == () and abs(float(norm) - want) <= 2.0 ** -24 * 1.01 * want
    factor = min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        u, step = torch.finfo(g.dtype).eps / 2, torch.finfo(g.dtype).tiny * torch.finfo(g.dtype).eps
        err = (g.double() - b.double() * factor).abs()
        assert bool((err <= (u + 2.01 * 2.0 ** -24) * (b.double() * factor).abs() + step / 2 * 1.01).all())
        if factor == 1.0:
            assert torch.equal(g, b)


def _grads(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtypes[i % len(dtypes)]).to(DEV) for i, s in enumerate(sizes)]


@pytest.mark.parametrize("dtypes", [[t] for t in TYPES] + [TYPES])
@pytest.mark.parametrize("sizes", [(1,), (7,), (8,), (4096,), (4097, 3), (1, 2, 3, 4, 5), (16384, 16385, 100003), (3, 0, 5), tuple(range(1, 170)),
                                   tuple(37 + i % 91 for i in range(500))])
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_norm_and_clip(sizes, dtypes, p):
    grads = _grads(sizes, dtypes, seed=len(sizes))
    assert abs(float(grad_norm(grads, p)) - _norm64(grads, p)) <= 2.0 ** -24 * 1.01 * _norm64(grads, p)
    _check_clip(grads, 0.25 * _norm64(grads, p), p)
    _check_clip(grads, 1e30, p)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", range(1, 8))
def test_views_at_every_element_and_nothing_beside_them(dtype, offset):
    """Gradients that start and end inside a 16-byte line: the neighbours keep their bits."""
    flat = _grads([400], [dtype], seed=offset)[0]
    before = flat.clone()
    grads = [flat[offset:offset + 5], flat[offset + 6:offset + 6 + 200], flat[offset + 300:offset + 301]]
    _check_clip(grads, 0.5)
    kept = torch.ones(400, dtype=torch.bool, device=DEV)
    for lo, hi in ((0, 5), (6, 206), (300, 301)):
        kept[offset + lo:offset + hi] = False
    assert torch.equal(flat[kept], before[kept])


def test_strided_gradients():
    g = _grads([64 * 3 * 3 * 32, 100 * 10, 40], [torch.float32])
    nhwc = g[0].view(64, 3, 3, 32).permute(0, 3, 1, 2)              # dense in another order
    cut = g[1].view(100, 10)[:, 2:7]                                # not dense: the columns beside it stay
    before = g[1].clone().view(100, 10)
    _check_clip([nhwc, cut, g[2]], 1.0)
    assert torch.equal(g[1].view(100, 10)[:, :2], before[:, :2]) and torch.equal(g[1].view(100, 10)[:, 7:], before[:, 7:])


def test_squares_beyond_fp32():
    """1e30 and 1e-30 squared leave fp32's range."""
    for scale in (1e30, 1e-30):
        grads = _grads([1000, 77], [torch.float32], scale=scale)
        assert abs(float(grad_norm(grads)) - _norm64(grads, 2)) <= 2.0 ** -23 * _norm64(grads, 2)
    _check_clip(_grads([1000, 77], [torch.float32], scale=1e30), 1.0)


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_non_finite(p, bad, dtype):
    grads = _grads([300, 5000], [dtype])
    grads[1][4321] = bad
    before = [g.clone() for g in grads]
    with pytest.raises(RuntimeError, match="not finite"):
        clip_grad_norm_(_params(grads), 1.0, p, error_if_nonfinite=True)
    assert all(torch.equal(a[a == a], b[a == a]) for a, b in zip(before, grads))
    norm = clip_grad_norm_(_params(grads), 1.0, p)
    if math.isnan(bad):
        assert math.isnan(float(norm)) and all(bool(g.isnan().all()) for g in grads)
    else:
        assert float(norm) == math.inf and bool(grads[1][4321].isnan()) and int(grads[0].count_nonzero()) == 0


def test_which_parameters_count():
    a, b = _grads([50, 60], [torch.float32])
    pa, pb = _params([a, b])
    none = torch.nn.Parameter(torch.zeros(5, device=DEV))
    want = _norm64([a, b], 2)
    assert abs(float(clip_grad_norm_([pa, none, pb, pa], 1e9)) - want) <= 2.0 ** -23 * want          # one that comes twice counts once
    assert float(clip_grad_norm_([none], 1.0)) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0 and float(grad_norm([])) == 0.0
    assert abs(float(clip_grad_norm_(pa, 1e9)) - _norm64([a], 2)) <= 2.0 ** -23 * want               # a lone tensor
    assert float(clip_grad_norm_(pa, 0.0)) > 0 and int(a.count_nonzero()) == 0                       # max_norm 0
    empty = torch.nn.Parameter(torch.zeros(0, device=DEV))
    empty.grad = torch.zeros(0, device=DEV)
    assert float(clip_grad_norm_([empty], 1.0)) == 0.0


def test_refusals():
    a = _grads([50], [torch.float32])[0]
    pa, pb = _params([a[:30], a[20:]])
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_([pa, pb], 1.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(RuntimeError, match="max_norm"):
            clip_grad_norm_([pa], bad)
    with pytest.raises(RuntimeError, match="fp16, bf16 or fp32"):
        grad_norm([a.double()])
    with pytest.raises(RuntimeError, match="type"):
        grad_norm([a], 3)
    with pytest.raises(RuntimeError, match="one device"):
        grad_norm([a, torch.zeros(3)])
    pe = torch.nn.Parameter(torch.zeros((4, 50), device=DEV))
    pe.grad = a.expand(4, 50)
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_([pe], 1.0)
    assert abs(float(grad_norm([pe.grad])) - 2 * _norm64([a], 2)) <= 2.0 ** -22 * _norm64([a], 2)
    pg = torch.nn.Parameter(torch.zeros(50, device=DEV))
    pg.grad = a * torch.nn.Parameter(torch.ones((), device=DEV))
    with pytest.raises(RuntimeError, match="graph"):
        clip_grad_norm_([pg], 1.0)


def test_same_gradients_same_bits():
    grads = _grads([100003, 77, 50000], TYPES)
    copies = [[g.clone() for g in grads] for _ in range(3)]
    norms = [clip_grad_norm_(_params(c), 1.0) for c in copies]
    assert all(torch.equal(norms[0], n) for n in norms) and all(torch.equal(x, y) for c in copies for x, y in zip(copies[0], c))


def test_captured_into_a_graph():
    """Two graphs and eager calls in turn: each replay clips what its gradients then hold."""
    lists = [_grads([5000, 33, 70000], TYPES, seed=s) for s in (1, 2)]
    values = [[g.clone() for g in grads] for grads in lists]
    params = [_params(grads) for grads in lists]
    graphs, norms = [], []
    for ps in params:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            clip_grad_norm_(ps, 1.0)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(clip_grad_norm_(ps, 1.0))
        graphs.append(g)
    for turn in range(3):
        for k in (0, 1):
            for g, v in zip(lists[k], values[k]):
                g.copy_(v * (turn + 1))
        for k in (0, 1):
            graphs[k].replay()
        for k in (0, 1):
            eager = [(v * (turn + 1)) for v in values[k]]
            n = clip_grad_norm_(_params(eager), 1.0)
            torch.cuda.synchronize()
            assert torch.equal(n, norms[k]) and all(torch.equal(a, b) for a, b in zip(eager, lists[k]))


# ------------------------------------------------------------------------------------------------------------ FusedSGD.step(max_norm)
def _model():
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Conv2d(3, 17, 3, bias=False), torch.nn.BatchNorm2d(17), torch.nn.Conv2d(17, 85, 1)).to(DEV)


@pytest.mark.parametrize("max_norm", [0.05, 1e9])
@pytest.mark.parametrize("scale", [None, 512.0])
@pytest.mark.parametrize("momentum", [0.937, 0.0])
def test_clipped_sgd_step(max_norm, scale, momentum):
    """Three steps against torch's clip_grad_norm_ + SGD in double precision.  Each step is off by a few fp32 roundings of its terms;
    three of them: 32 * 2^-24 of the largest."""
    model = _model()
    ref = [p.detach().double().clone().requires_grad_() for p in model.parameters()]
    arena = ParamArena(model)
    opt = FusedSGD(model, arena, lr=0.1, momentum=momentum, nesterov=momentum > 0)
    kinds = [opt.group[arena.offset_of(p)].item() for p in model.parameters()]
    topt = torch.optim.SGD([{"params": [r], "weight_decay": 5e-4 if k == 1 else 0.0} for r, k in zip(ref, kinds)], lr=0.1, momentum=momentum,
                           nesterov=momentum > 0)
    scaler = LossScaler(DEV, init_scale=scale) if scale else None
    g = torch.Generator().manual_seed(5)
    for step in range(3):
        for p, r in zip(model.parameters(), ref):
            v = torch.randn(p.shape, generator=g).to(DEV) * 0.01
            p.grad.copy_(v * (scale or 1.0))
            r.grad = v.double() * 0.5
        kept = arena.grad.clone()
        norm = opt.step(scaler, grad_mul=0.5, max_norm=max_norm)
        want = torch.nn.utils.clip_grad_norm_(ref, max_norm)
        topt.step()
        assert abs(float(norm) - float(want)) <= 2.0 ** -22 * float(want)
        assert torch.equal(arena.grad, kept)                        # the factor lives in the update
    for p, r in zip(model.parameters(), ref):
        assert float((p.detach().double() - r.detach()).abs().max()) <= 32 * 2.0 ** -24 * max(1.0, float(r.detach().abs().max()))


def test_clipped_step_without_clipping_is_the_step():
    """Gradients below max_norm: the bits of the step without it."""
    models = [_model(), _model()]
    arenas = [ParamArena(m) for m in models]
    opts = [FusedSGD(m, a) for m, a in zip(models, arenas)]
    for step in range(3):
        g = torch.Generator().manual_seed(step)
        v = torch.randn(arenas[0].numel, generator=g).to(DEV) * 0.01
        for a in arenas:
            a.grad.copy_(v)
        assert opts[0].step() is None
        opts[1].step(max_norm=1e9)
    assert torch.equal(arenas[0].data, arenas[1].data) and torch.equal(opts[0].buf, opts[1].buf)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_clipped_step_skips_on_overflow(bad):
    model = _model()
    arena = ParamArena(model)
    opt, scaler = FusedSGD(model, arena), LossScaler(DEV, init_scale=64.0)
    arena.grad.normal_()
    opt.step(scaler, max_norm=1.0)
    data, buf = arena.data.clone(), opt.buf.clone()
    arena.grad[7] = bad
    norm = opt.step(scaler, max_norm=1.0)
    assert not math.isfinite(float(norm)) and int(scaler.found_inf) == 1
    assert torch.equal(arena.data, data) and torch.equal(opt.buf, buf)
    scaler.update()
    assert float(scaler.scale) == 32.0 and int(scaler.found_inf) == 0
    arena.grad.normal_()
    scaler.found_inf.fill_(1)                                       # another check's flag counts too
    opt.step(scaler, max_norm=1.0)
    assert torch.equal(arena.data, data)


def test_a_gradient_of_more_than_2_to_the_30_elements():
    """Several entries of one tensor, offsets past 32 bits: constant values, so that the sums are known."""
    n = (1 << 31) + 5
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device=DEV)
    g[-1] = 4.0
    want = math.sqrt(0.25 * (n - 1) + 16.0)
    assert abs(float(grad_norm([g])) - want) <= 2.0 ** -23 * want
    norm = clip_grad_norm_(_params([g[3:]]), 1.0)
    want = math.sqrt(0.25 * (n - 4) + 16.0)
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    small = torch.tensor(0.5 / want, dtype=torch.float64).to(torch.bfloat16)
    assert bool((g[:3] == 0.5).all())
    for lo in range(3, n - 1, 1 << 28):
        part = g[lo:min(lo + (1 << 28), n - 1)]
        assert float((part.float() - float(small)).abs().max()) <= 2.0 ** -8 * float(small)
    assert abs(float(g[-1]) - 4.0 / want) <= 2.0 ** -8 * 4.0 / want


def test_gradients_with_gaps():
    """Columns of one buffer, interleaved: each is scaled; the same columns twice are refused and left as they were."""
    from yolov6_amd.solver import clip_grad_norm_
    buf = torch.randn(64, 10, device="cuda")
    before = buf.clone()
    params = [torch.nn.Parameter(torch.zeros(64, 5, device="cuda")) for _ in range(2)]
    params[0].grad, params[1].grad = buf[:, ::2], buf[:, 1::2]
    norm = clip_grad_norm_(params, 0.5)
    want = before.double().norm()
    assert abs(float(norm) - float(want)) <= 2 * 2.0 ** -24 * float(want)
    assert torch.allclose(buf.double(), before.double() * (0.5 / (want + 1e-6)), rtol=4 * 2.0 ** -24, atol=0)
    before = buf.clone()
    params[1].grad = buf[:, ::2]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_(params, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(buf, before)


def test_forward_mode_is_refused():
    g = _grads([50], [torch.float32])[0]
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(g, torch.ones_like(g))
        with pytest.raises(RuntimeError, match="forward mode"):
            grad_norm([dual])


def test_clipping_counts_as_a_write():
    """Autograd sees it: version counters of dense gradients and of ones with gaps go up, a graph that saved one refuses its backward."""
    buf = torch.randn(64, 10, device=DEV)
    params = _params([_grads([500], [torch.float32])[0], _grads([77], [torch.float16])[0], buf[:, ::2]])
    before = [p.grad._version for p in params]
    grad_norm([p.grad for p in params])
    assert [p.grad._version for p in params] == before
    w = torch.ones(500, device=DEV, requires_grad=True)
    y = (w * params[0].grad).sum()
    clip_grad_norm_(params, 1.0)
    assert all(p.grad._version > v for p, v in zip(params, before))
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        held = torch.nn.Parameter(torch.zeros(9, device=DEV), requires_grad=False)
        held.grad = torch.full((9,), 2.0, device=DEV)
        assert abs(float(clip_grad_norm_([held], 1.0)) - 6.0) <= 6 * 2.0 ** -23


def test_gradients_with_gaps_that_share_a_part():
    """Those that start apart are not told from ones that share nothing: each element is scaled once, the norm counts each gradient whole."""
    buf = torch.randn(64, 10, device=DEV)
    before = buf.double()
    params = _params([buf[:, :6], buf[:, 4:9], buf[:, 9:]])
    want = math.sqrt(float(before.square().sum() + before[:, 4:6].square().sum()))
    norm = clip_grad_norm_(params, 0.5)
    assert abs(float(norm) - want) <= 2 * 2.0 ** -24 * want
    assert torch.allclose(buf.double(), before * (0.5 / (want + 1e-6)), rtol=4 * 2.0 ** -24, atol=0)


def test_a_step_over_nothing_has_norm_zero():
    import ctypes as C
    from yolov6_amd import _lib
    lib = _lib.load()
    buf, norm = torch.ones(64, device=DEV), torch.full((), 7.0, device=DEV)
    at = C.c_void_p(buf.data_ptr())
    three = (C.c_float * 3)(0.1, 0.1, 0.1)
    _lib.check(lib.y6_sgd_step_clipped(at, at, at, at, 0, three, three, 0.9, 1, 0, 1.0, None, None, 1.0, at, 256, C.c_void_p(norm.data_ptr()),
                                       _lib.current_stream_ptr()), "sgd_step_clipped")
    torch.cuda.synchronize()
    assert float(norm) == 0.0 and bool((buf == 1).all())
