"""pir_amd.optim on the GPU: every type, layout and size against 64 bits, graphs, streams, offsets past 32 bits, and a
training run on the kernels."""
import functools
import math

import pytest
import torch

import optim_util as U
from pir_amd import optim, train
from test_optim import LAYOUTS, assert_moved_alike, check_load_of_another_order, networks, optimizer_of, overlaps, refused_call, run, train_steps

pytestmark = pytest.mark.gpu
DEV = "cuda"
SIZES = [0, 1, 2, 3, 4, 5, 7, 8, 63, 64, 65, 255, 256, 257, 511, 513, 1023, 4095, 4096, 4097, 10_007, 70_001]


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", U.TYPES)
def test_step_matches_64_bits(dtype, bits, odd):
    U.check_step(run, SIZES, dtype, bits, DEV, odd=odd)


@pytest.mark.parametrize("max_norm", [1e-3, 0.2, 100.0, math.inf])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", U.TYPES)
def test_clipped_step_matches_64_bits(dtype, bits, max_norm):
    U.check_step(run, SIZES[1:], dtype, bits, DEV, odd=True, max_norm=max_norm, seed=4)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 63, 64, 65, 130, 192, 193, 400, 600])
def test_any_number_of_tensors(count, bits):
    U.check_step(run, [1 + (37 * i) % 700 for i in range(count)], torch.float32, bits, DEV, odd=True, max_norm=0.1, seed=count)


@pytest.mark.parametrize("hyper", [
    dict(lr=0.0, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1), dict(lr=1e-2, betas=(0.0, 0.0), eps=1e-8, weight_decay=0.0),
    dict(lr=1e-4, betas=(0.99, 0.9999), eps=1e-3, weight_decay=1.0), dict(lr=0.5, betas=(0.5, 0.1), eps=1.0, weight_decay=0.3)])
@pytest.mark.parametrize("bits", [32, 8])
def test_hyper_parameters(hyper, bits):
    U.check_step(run, [5, 300, 5000], torch.float32, bits, DEV, hyper=hyper)


@pytest.mark.parametrize("scale", [1e-12, 1e6])
@pytest.mark.parametrize("bits", [32, 8])
def test_sizes_of_gradients(scale, bits):
    U.check_step(run, [5, 300, 5000], torch.float32, bits, DEV, scale=scale,
                 hyper=dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8 * min(1.0, scale), weight_decay=0.0))


@pytest.mark.parametrize("bits", [32, 8])
def test_step_counts_from_the_first_to_late_ones(bits):
    """1 - beta2^t at t = 1 loses three digits where beta is rounded to fp32 first."""
    p, g, m, v, s, steps = U.make([300] * 6, torch.float32, bits, DEV)
    counts = [0.0, 1.0, 10.0, 1e3, 1e5, 2.0 ** 24 - 1]
    steps.copy_(torch.tensor(counts))
    keep = [[t.clone() for t in x] if x is not None else None for x in (p, g, m, v, s)]
    hyper = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    run(p, g, m, v, s, steps, None, **hyper)
    for i, t in enumerate(counts):
        old = (keep[2][i], keep[3][i], keep[4][i]) if bits == 8 else keep[2][i]
        want, bound = U.step64(keep[0][i], keep[1][i], old, keep[3][i], t + 1, **hyper)
        U.assert_near(p[i], want[0], bound[0], f"after step {t + 1:g}")


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts(bits):
    """Transposed parameters keep their order of memory; gradients in another order, expanded or with gaps are taken by
    value."""
    gen = torch.Generator().manual_seed(0)
    rand = lambda *n: torch.randn(*n, generator=gen).to(DEV)  # noqa: E731
    p = [rand(40, 30).t(), rand(6, 5, 4).permute(1, 2, 0), rand(30, 40), rand(7, 1), rand(())]
    g = [rand(30, 40), rand(5, 4, 6), rand(40, 30).t(), rand(1, 1).expand(7, 1), rand(())]
    g.append(rand(25, 2)[:, 0])
    p.append(rand(25))
    steps = torch.zeros(len(p), device=DEV)
    keep = [t.clone() for t in p]
    m = [torch.zeros_like(t) for t in p]
    v = [torch.zeros_like(t) for t in p]
    s = None
    if bits == 8:
        m, v, s = zip(*(optim.moments8_encode(a, b) for a, b in zip(m, v)))
    hyper = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    run(p, g, list(m), list(v), s, steps, None, **hyper)
    for i, (a, b, c) in enumerate(zip(p, keep, g)):
        z = torch.zeros_like(c).contiguous()
        want, bound = U.step64(b.contiguous(), c.contiguous(), z, z, 1, **hyper)
        U.assert_near(a.contiguous(), want[0], 2 * bound[0], f"layout {i}")


@pytest.mark.parametrize("dtype", U.TYPES)
@pytest.mark.parametrize("numel", [1, 255, 256, 257, 10_007, 1_000_003])
def test_moments8_both_ways(numel, dtype):
    gen = torch.Generator().manual_seed(numel)
    m = (torch.randn(numel, generator=gen) * torch.exp(2 * torch.randn(numel, generator=gen))).to(dtype)
    v = (torch.rand(numel, generator=gen) * torch.exp(2 * torch.randn(numel, generator=gen))).to(dtype)
    q, c, s = optim.moments8_encode(m.to(DEV), v.to(DEV))
    U.assert_coded(q, c, s, m.double(), v.double(), 2 * U.E * m.double().abs(), 2 * U.E * v.double(), "encode")
    assert bool((q.view(-1)[numel:] == 0).all()) and bool((c.view(-1)[numel:] == 0).all())
    a, b = optim.moments8_decode(q, c, s, dtype=dtype)
    x, y = U.decode64(q, c, s)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half if dtype == torch.float16 else 0.0   # below: steps of its subnormals
    fits = y.reshape(-1) < torch.finfo(dtype).max
    U.assert_near(a, x.reshape(-1), ((half + 6 * U.E) * x.abs() + tiny).reshape(-1), "decoded m")
    U.assert_near(b.reshape(-1)[fits.to(DEV)], y.reshape(-1)[fits], ((half + 12 * U.E) * y.abs() + tiny).reshape(-1)[fits], "decoded v")


def test_moments8_special_blocks():
    m, v = torch.ones(6 * 256), torch.ones(6 * 256)
    m[:256], v[:256] = 0.0, 0.0
    m[256:512] = 1e-39
    m[512 + 7], v[768 + 9], m[1024], m[1280:], v[1280:] = math.inf, math.nan, -math.inf, 3e38, 3e38
    got = [optim.moments8_encode(x.to(DEV), y.to(DEV)) for x, y in ((m, v),)][0]
    want = optim.moments8_encode(m, v)
    assert torch.equal(got[2].isnan().cpu(), want[2].isnan()) and torch.equal(got[2].cpu().nan_to_num(), want[2].nan_to_num())
    a, b = optim.moments8_decode(*got)
    assert float(a[0].abs().max()) == 0 and float(b[0].max()) == 0 and float(a[1].abs().max()) == 0
    assert bool(a[2].isnan().all()) and bool((b[2] == 1).all()) and bool(b[3].isnan().all()) and bool(a[4].isnan().all())
    for x in (a, b):
        assert float((x[5] / 3e38 - 1).abs().max()) < 1e-6


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(bits):
    """In 32 bits they ruin their own element; in 8 the moments of their block.  Other blocks never see them."""
    p, g, m, v, s, steps = U.make([1000, 256], torch.float32, bits, DEV)
    keep = [x.clone() for x in p]
    g[0][300], g[0][700] = math.nan, math.inf
    run(p, g, m, v, s, steps, None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    bad = torch.zeros(1000, dtype=torch.bool, device=DEV)
    bad[300] = bad[700] = True
    assert torch.equal(~p[0].isfinite(), bad) and bool(p[1].isfinite().all())
    if bits == 8:
        assert s[0].isnan().any(1).tolist() == [False, True, True, False] and not bool(s[1].isnan().any())
    else:
        assert torch.equal(~m[0].isfinite(), bad)
    # and where the step is to be skipped, nothing moves, the counts included
    p, g, m, v, s, steps = U.make([1000, 256], torch.float32, bits, DEV)
    g[0][300] = math.nan
    all_of = lambda: [x.clone() for y in (p, m, v, s or []) for x in y] + [steps.clone()]  # noqa: E731
    before = all_of()
    norm = optim._step(p, g, m, v, s, steps, 1e-3, (0.9, 0.999), 1e-8, 0.0, 1.0, True)
    assert math.isnan(float(norm)) and all(torch.equal(a, b) for a, b in zip(before, all_of()))
    g[0][300] = 0.0
    optim._step(p, g, m, v, s, steps, 1e-3, (0.9, 0.999), 1e-8, 0.0, 1.0, True)
    assert torch.equal(steps, before[-1] + 1) and not torch.equal(p[0], keep[0])


@pytest.mark.parametrize("device", ["cpu", DEV])
def test_scales_of_moments_that_are_not_finite(device):
    """A second moment past fp32's largest takes both scales of its block with it; a first moment's scale that is NaN stays
    so, and says nothing about other blocks."""
    p, g, m, v, s, steps = U.make([1024], torch.float32, 8, device)
    g[0][300] = 1e21                                     # 0.001 1e42
    s[0][2, 0] = math.nan
    run(p, g, m, v, s, steps, None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    assert s[0].isnan().tolist() == [[False, False], [True, True], [True, False], [False, False]]
    assert p[0].isnan().nonzero().view(-1).tolist() == list(range(512, 768))


def test_blocks_without_gradients_keep_their_parameters():
    """Moments of zero and gradients of zero: no step, and 0 / (0 + eps) is no NaN; a block that then gets one starts."""
    p = [torch.randn(600, device=DEV)]
    g = [torch.zeros(600, device=DEV)]
    q, c, s = optim.moments8_encode(torch.zeros(600, device=DEV), torch.zeros(600, device=DEV))
    steps = torch.zeros(1, device=DEV)
    keep = p[0].clone()
    for _ in range(3):
        optim.adamw8_step(p, g, [q], [c], [s], steps, lr=1e-3)
    assert torch.equal(p[0], keep)
    g[0][300] = 1e-3
    optim.adamw8_step(p, g, [q], [c], [s], steps, lr=1e-3)
    moved = p[0] != keep
    assert int(moved.sum()) == 1 and bool(moved[300])


@pytest.mark.parametrize("dtype", U.TYPES)
def test_grad_norm(dtype):
    gen = torch.Generator().manual_seed(3)
    g = [(0.01 * torch.randn(n + 1, generator=gen)).to(dtype).to(DEV)[1:] for n in SIZES + [16_383, 16_384, 16_385, 300_000]]
    total, each = optim.grad_norm(g)
    want = [math.sqrt(float(x.double().square().sum())) for x in g]
    assert total.dtype == torch.float32 and total.dim() == 0 and each.shape == (len(g),)
    # sums in 64 bits: n 2^-53 at most, then one rounding to fp32
    assert abs(float(total) - U.norm64(g)) <= 1.001 * U.E * U.norm64(g)
    for a, b in zip(each.tolist(), want):
        assert abs(a - b) <= 1.001 * U.E * b
    again = optim.grad_norm(g)
    assert torch.equal(total, again[0]) and torch.equal(each, again[1])


@pytest.mark.parametrize("count", [1, 64, 65, 312, 313, 511, 512, 513, 1100])
def test_grad_norm_of_many(count):
    g = [torch.full((1 + i % 5,), float(i), device=DEV) for i in range(count)]
    total, each = optim.grad_norm(g)
    want = [i * math.sqrt(1 + i % 5) for i in range(count)]
    assert all(abs(a - b) <= 1.001 * U.E * b for a, b in zip(each.tolist(), want))
    all_of = math.sqrt(math.fsum(x * x for x in want))
    assert abs(float(total) - all_of) <= 1.001 * U.E * all_of


def test_grad_norm_of_the_largest_and_smallest_values():
    big, small = torch.full((1000,), 3e37, device=DEV), torch.full((1000,), 1e-37, device=DEV)
    # sqrt(1000) 3e37 = 9.5e38 is past fp32's largest, 3.4e38: its rounding to fp32 is infinity; of a hundred of them it fits
    assert float(optim.grad_norm([big])[0]) == math.inf
    for g, want in ((big[:100], 3e37 * 10), (small, 1e-37 * math.sqrt(1000))):
        assert abs(float(optim.grad_norm([g])[0]) / want - 1) < 1e-6     # the values themselves are rounded to fp32
    assert float(optim.grad_norm([torch.tensor([1.0, math.inf], device=DEV)])[0]) == math.inf
    assert math.isnan(float(optim.grad_norm([torch.tensor([1.0, math.nan], device=DEV)])[0]))
    assert float(optim.grad_norm([torch.zeros(0, device=DEV), torch.zeros(9, device=DEV)])[0]) == 0.0
    t = torch.randn(64, 48, device=DEV)
    assert float(optim.grad_norm([t.t()])[0]) == float(optim.grad_norm([t])[0])
    assert abs(float(optim.grad_norm([t[:, ::2]])[0]) - float(t[:, ::2].double().norm())) < 1e-5


@pytest.mark.parametrize("bits", [32, 8])
def test_same_bits_on_every_run(bits):
    got = []
    for _ in range(2):
        p, g, m, v, s, steps = U.make([70_001, 513, 9], torch.bfloat16, bits, DEV)
        for _ in range(3):
            run(p, g, m, v, s, steps, 0.1, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
        got.append([t.clone() for x in (p, m, v, s or []) for t in x])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_mixed_types_and_moments_in_one_call():
    """One joint norm over fp32, bf16 and fp16 parameters, some with moments in 8 bits, groups with their own settings."""
    sizes = [(torch.float32, 5000), (torch.bfloat16, 70_000), (torch.float16, 300), (torch.float32, 100), (torch.bfloat16, 0), (torch.bfloat16, 257)]
    gen = torch.Generator().manual_seed(8)
    ps = [torch.nn.Parameter((0.05 * torch.randn(n, generator=gen)).to(t).to(DEV)) for t, n in sizes]
    groups = [{"params": ps[:2], "lr": 1e-3, "state_bits": 8}, {"params": ps[2:4], "lr": 1e-2, "weight_decay": 0.3, "betas": (0.8, 0.9)},
              {"params": ps[4:], "state_bits": 8, "min_8bit_numel": 1}]
    opt = optim.AdamW(groups, lr=1e-4, weight_decay=0.01, max_norm=0.05)
    twins = [p.detach().clone() for p in ps]
    for p in ps:
        p.grad = (1e-2 * torch.randn(p.shape, generator=gen)).to(p.dtype).to(DEV)
    opt.step()
    total = U.norm64([p.grad for p in ps])
    assert abs(float(opt.total_norm) - total) <= 1.001 * U.E * total
    for i, (p, q) in enumerate(zip(ps, twins)):
        g = opt.param_groups[0 if i < 2 else 1 if i < 4 else 2]
        z = torch.zeros(p.numel())
        want, bound = U.step64(q, p.grad, z, z, 1, g["lr"], g["betas"], g["eps"], g["weight_decay"], 0.05 / (total + 1e-6))
        U.assert_near(p, want[0], bound[0], f"parameter {i}")
        assert ("scales" in opt.state[p]) == (i in (0, 1, 5))


@pytest.mark.parametrize("max_norm", [None, 1e3])
def test_more_groups_than_one_prologue_holds(max_norm):
    ps = [torch.nn.Parameter(torch.ones(5, device=DEV)) for _ in range(40)]
    opt = optim.AdamW([{"params": [p], "lr": 1e-3 * (i + 1)} for i, p in enumerate(ps)], weight_decay=0.0, max_norm=max_norm)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    for i, p in enumerate(ps):                           # first step: lr times the sign of the gradient
        assert float((1 - p.detach() - 1e-3 * (i + 1)).abs().max()) < 2e-7
    assert all(float(opt.state[p]["step"]) == 1 for p in ps)


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_far_apart(bits):
    """More than 8 GB between two tensors of a call, in either order: descriptors are differences of 32 bits."""
    room = torch.empty(20 * 2 ** 30, dtype=torch.uint8, device=DEV).view(torch.float32)
    hyper = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    p, g, m, v, s, steps = U.make([5000] * 4, torch.float32, bits, DEV)
    away = [room[i + 10_000:i + 15_000].copy_(x) for i, x in zip((0, room.numel() - 25_000, 5000, room.numel() // 2), g)]
    for x, y in zip(optim.grad_norm(away), optim.grad_norm(g)):
        assert torch.equal(x, y)
    near = [t.clone() for t in p], g, [t.clone() for t in m], [t.clone() for t in v], None if s is None else [t.clone() for t in s], steps.clone()
    at = [room.numel() - 5000, 0, room.numel() // 2, 5000]
    far = [room[i:i + 5000].copy_(t) for i, t in zip(at, p)]
    run(far, away, m, v, s, steps, 0.1, **hyper)
    run(*near, 0.1, **hyper)
    assert all(torch.equal(a, b) for a, b in zip(far, near[0])) and torch.equal(steps, near[5])
    assert all(torch.equal(a, b) for a, b in zip(m, near[2])) and all(torch.equal(a, b) for a, b in zip(v, near[3]))


@pytest.mark.parametrize("bits", [32, 8])
def test_skipped_step_of_many_tensors(bits):
    p, g, m, v, s, steps = U.make([40] * 300, torch.float32, bits, DEV)
    before = [x.clone() for y in (p, m, v, s or []) for x in y] + [steps.clone()]
    g[299][39] = -math.inf
    norm = optim._step(p, g, m, v, s, steps, 1e-3, (0.9, 0.999), 1e-8, 0.0, None, True)
    assert float(norm) == math.inf and all(torch.equal(a, b) for a, b in zip(before, [x for y in (p, m, v, s or []) for x in y] + [steps]))


def test_first_step_is_not_captured(monkeypatch):
    w = torch.nn.Parameter(torch.ones(9, device=DEV))
    w.grad = torch.ones_like(w)
    opt = optim.AdamW([w])
    with monkeypatch.context() as patch:
        patch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
    opt.step()
    assert float(opt.state[w]["step"]) == 1


def test_captured_step_of_the_class():
    """A first step, the capture, replays with an eager step between them: as many eager steps."""
    nets = [networks().to(DEV) for _ in range(2)]
    opts = [optim.AdamW(n.parameters(), lr=1e-3, state_bits=8, min_8bit_numel=256, max_norm=1e-2) for n in nets]
    x = torch.randn(32, 3, generator=torch.Generator().manual_seed(0)).to(DEV)
    for net, opt in zip(nets, opts):
        net(x).square().mean().backward()
        opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()                                   # records the step, runs nothing
    for k in range(4):
        for net in nets:
            for p in net.parameters():
                p.grad.mul_(1.1)
        graph.replay() if k != 2 else opts[0].step()
        opts[1].step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(nets[0].parameters(), nets[1].parameters())), k


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed(bits):
    """A captured step is a step at every replay: the counts move on, the learning rate is read on the device, and eager
    steps between the replays take their turn."""
    sizes = [70_001, 300, 5]
    a, b = U.make(sizes, torch.float32, bits, DEV), U.make(sizes, torch.float32, bits, DEV)
    lr = torch.tensor(1e-3, device=DEV)
    hyper = dict(betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    call = lambda x, rate: run(*x, 0.05, lr=rate, **hyper)  # noqa: E731
    norms = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(a, lr)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(a, lr)
    call(b, lr)
    gen = torch.Generator().manual_seed(5)
    for k in range(6):
        new = [(1e-3 * torch.randn(n, generator=gen)).to(DEV) for n in sizes]
        lr.fill_(1e-3 / (k + 1))
        for x in (a, b):
            for g, n in zip(x[1], new):
                g.copy_(n)
        if k == 3:
            call(a, lr)
        else:
            graph.replay()
            norms.append(float(out))
        want = call(b, float(lr))
        assert k == 3 or norms[-1] == float(want)
        torch.cuda.synchronize()
        for x, y in zip(a, b):
            if x is not None:
                assert all(torch.equal(i, j) for i, j in zip(x, y)), k
    assert a[5].tolist() == [3.0 + i % 3 + 7 for i in range(3)]


def test_two_graphs_side_by_side():
    """Two captured steps share no workspace: replayed together on two streams they give what they give alone."""
    sets = [U.make([300_000, 17], torch.float32, bits, DEV, seed=bits) for bits in (32, 8)]
    alone = [U.make([300_000, 17], torch.float32, bits, DEV, seed=bits) for bits in (32, 8)]
    hyper = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    graphs = []
    for s in sets:
        run(*s, 0.05, **hyper)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(*s, 0.05, **hyper)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, t in zip(sets, alone):
        for _ in range(6):
            run(*t, 0.05, **hyper)
        for x, y in zip(s, t):
            if x is not None:
                assert all(torch.equal(i, j) for i, j in zip(x, y))


def test_one_optimizer_on_two_devices():
    ps = [torch.nn.Parameter(torch.ones(300)), torch.nn.Parameter(torch.ones(300, device=DEV))]
    opt = optim.AdamW(ps, lr=1e-2, weight_decay=0.0)
    for p in ps:
        p.grad = torch.full_like(p, 0.5)
    opt.step()
    assert all(float((1 - p.detach() - 1e-2).abs().max()) < 2e-7 for p in ps)
    with pytest.raises(ValueError, match="several devices"):
        optim.step_together([opt], max_norm=1.0)


def test_c_calls_with_the_least():
    """A norm without those of each, a norm of nothing, a step of nothing that is asked for its norm."""
    import ctypes
    from pir_amd import _lib
    L, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    g = torch.full((10_000,), 2.0, device=DEV)
    out, work = torch.full((3,), -1.0, device=DEV), torch.empty(1 << 16, dtype=torch.uint8, device=DEV)
    grads, numels, dtypes = (ctypes.c_void_p * 1)(g.data_ptr()), (ctypes.c_long * 1)(10_000), (ctypes.c_int * 1)(0)
    at = [ctypes.addressof(x) for x in (grads, numels, dtypes)]
    assert L.pir_grad_norm(1, *at, out.data_ptr(), None, work.data_ptr(), work.numel(), stream) == 0
    assert L.pir_grad_norm(0, *at, out.data_ptr() + 4, None, work.data_ptr(), work.numel(), stream) == 0
    assert L.pir_adamw_step(0, *[None] * 10, 0, 0.0, 0, out.data_ptr() + 8, work.data_ptr(), work.numel(), stream) == 0
    assert out.tolist() == [200.0, 0.0, 0.0]


@pytest.mark.parametrize("bits", [32, 8])
def test_empty_tensors_alone(bits):
    U.check_step(run, [0], torch.float32, bits, DEV)
    U.check_step(run, [0, 0, 300, 0], torch.bfloat16, bits, DEV, max_norm=1.0)


def test_another_stream():
    p, g, m, v, s, steps = U.make([300_000], torch.float32, 32, DEV)
    q = [t.clone() for t in p], g, [t.clone() for t in m], [t.clone() for t in v], None, steps.clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    hyper = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    with torch.cuda.stream(st):
        for _ in range(3):
            run(p, g, m, v, s, steps, 0.1, **hyper)
    torch.cuda.current_stream().wait_stream(st)
    for _ in range(3):
        run(*q, 0.1, **hyper)
    assert torch.equal(p[0], q[0][0]) and torch.equal(v[0], q[3][0])


def test_versions_move_on():
    """Autograd and the networks' packed weights go by the version of a parameter."""
    w = torch.nn.Parameter(torch.randn(10, device=DEV))
    y = (w * w).sum()
    opt = optim.AdamW([w])
    w.grad = torch.ones_like(w)
    before = w._version
    opt.step()
    assert w._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    from gpu_util import sdf_net
    net = sdf_net("sdf_full.npz")
    x = torch.randn(100, 3, device=DEV) * 0.5
    with torch.no_grad():
        first = net.sdf(x)
    opt = optim.AdamW(net.parameters(), lr=1e-2)
    net.sdf(x).square().sum().backward()
    opt.step()
    from pir_amd.network import invalidate_packed
    with torch.no_grad():
        second = net.sdf(x)
        invalidate_packed(net)
        third = net.sdf(x)
    assert not torch.equal(first, second) and torch.equal(second, third)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("source", ["torch", 32, 8])
def test_class_against_torch_and_its_checkpoints(source, bits):
    net = networks().to(DEV)
    start = [p.detach().clone() for p in net.parameters()]
    make = lambda n, b: torch.optim.Adam(n.parameters(), lr=1e-3) if b == "torch" else \
        optim.AdamW(n.parameters(), lr=1e-3, weight_decay=0.0, state_bits=b, min_8bit_numel=100)  # noqa: E731
    steps = functools.partial(train_steps_on, DEV)
    first = make(net, source)
    steps(net, first, 4)
    other = networks().to(DEV)
    other.load_state_dict(net.state_dict())
    second = make(other, bits)
    saved = first.state_dict()
    second.load_state_dict({**saved, "param_groups": [{**saved["param_groups"][0], "state_bits": bits, "min_8bit_numel": 100}]})
    steps(net, first, 1, seed=9)
    steps(other, second, 1, seed=9)
    assert_moved_alike(net, other, start, 1e-3, 1, part=1e-3 if source != 8 and bits == 32 or source == bits else 0.3)


def train_steps_on(device, net, opt, steps, seed=0):
    gen = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        opt.zero_grad()
        x = torch.randn(32, 3, generator=gen).to(device)
        ((net(x) - x.sum(1, keepdim=True)) ** 2).mean().backward()
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_past_32_bits(bits):
    """2^31 + 777 bf16 elements in one tensor: its head and its tail are what the same elements give in tensors of their
    own, and the norm counts all of them."""
    n, k = 2 ** 31 + 777, 5 * 256
    tail = n - (n - k) // 256 * 256                      # whole blocks, counted from the front
    p = torch.full((n,), 0.5, dtype=torch.bfloat16, device=DEV)
    g = torch.full((n,), 2.0 ** -10, dtype=torch.bfloat16, device=DEV)
    gen = torch.Generator().manual_seed(1)
    ends = [slice(0, k), slice(n - tail, n)]
    for e in ends:
        p[e] = (0.05 * torch.randn(e.stop - e.start, generator=gen)).bfloat16().to(DEV)
        g[e] = (1e-3 * torch.randn(e.stop - e.start, generator=gen)).bfloat16().to(DEV)
    small = [p[e].clone() for e in ends], [g[e].clone() for e in ends]
    hyper = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)

    def state(n):
        if bits == 32:
            return torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), None
        nb = -(-n // 256)
        return (torch.zeros(nb, 256, dtype=torch.int8, device=DEV), torch.zeros(nb, 256, dtype=torch.uint8, device=DEV),
                torch.zeros(nb, 2, device=DEV))
    m, v, s = state(n)
    total, _ = optim.grad_norm([g])
    want = math.sqrt((n - k - tail) * 2.0 ** -20 + U.norm64(small[1]) ** 2)
    assert abs(float(total) - want) <= 2 * U.E * want
    run([p], [g], [m], [v], None if s is None else [s], torch.zeros(1, device=DEV), None, **hyper)
    m2, v2, s2 = zip(*(state(x.numel()) for x in small[0]))
    run(*small, list(m2), list(v2), None if s is None else list(s2), torch.zeros(2, device=DEV), None, **hyper)
    for i, e in enumerate(ends):
        assert torch.equal(p[e], small[0][i])
        if bits == 32:
            assert torch.equal(m[e], m2[i]) and torch.equal(v[e], v2[i])
        else:
            rows = slice(e.start // 256, -(-e.stop // 256))
            assert torch.equal(m[rows], m2[i]) and torch.equal(v[rows], v2[i]) and torch.equal(s[rows], s2[i])
    mid = p[k:n - tail]
    assert bool((mid == mid[0]).all()) and float(mid[0]) != 0.5


@pytest.mark.parametrize("kind", ["adamw", "adamw8"])
def test_training_trajectory_on_the_kernels(kind, monkeypatch):
    """Five iterations of the training loop with this package's optimizers, all networks in one step: the reference's losses
    and masks; in 32 bits its parameters too (as in the trajectory test with torch.optim.Adam)."""
    import train_traj_util
    monkeypatch.setattr(train, "make_optimizers", functools.partial(train.make_optimizers, optimizer=kind))
    tol = (0.06, 0.6) if kind == "adamw" else (0.2, 1.5)  # 8 bits: percents of a step of lr, over five of them
    out = train_traj_util.run("cuda", loss_tol=1e-3, exact_masks=False, step_tol=tol)
    assert len(out["losses"]) >= 2


def test_training_step_clips_the_joint_norm():
    import numpy as np
    import train_step_util
    d, state = train_step_util.build_state("cuda")
    lr = dict(sdf_network=1e-5, dino_network=1e-3, **{k: 1e-4 for k in state.color_network_dict})
    state.sdf_optimizer, state.color_optimizer_dict, state.dino_optimizer = train.make_optimizers(
        state.sdf_network, state.color_network_dict, state.dino_network, lr, True, optimizer="adamw")
    state.max_grad_norm = 1e-3
    np.random.seed(int(d["np_seed"]))
    torch.manual_seed(0)
    before = [p.detach().clone() for p in state.sdf_network.parameters()]
    out = train.training_step(state, 12000)
    ps = [p for p in list(state.sdf_network.parameters()) + list(state.color_network_dict["point_light_network"].parameters())
          if p.grad is not None]
    want = U.norm64([p.grad for p in ps])
    assert abs(out["grad_norm"] - want) <= 1.001 * U.E * want
    opt = state.sdf_optimizer
    for p, q in zip(state.sdf_network.parameters(), before):
        if p.grad is None:
            continue
        bound = 6 * U.E * 0.1 * p.grad.double().abs() * 1e-3 / want + 1e-44
        assert bool(((opt.state[p]["exp_avg"] - 0.1 * p.grad.double() * min(1.0, 1e-3 / (want + 1e-6))).abs() <= bound).all())
        assert not torch.equal(p, q)


@pytest.mark.parametrize("bits, what", [(b, w) for b in (32, 8) for w in overlaps(b)])
def test_overlapping_tensors_are_refused(bits, what):
    refused_call(bits, what, DEV)


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_in_any_order_of_memory(bits):
    """Lists whose tensors lie among each other in one buffer, backwards, gradients shared: what the same values give in
    tensors of their own."""
    n, k = 1024, 12
    gen = torch.Generator().manual_seed(2)
    values = torch.randn(2, k, n, generator=gen).to(DEV)
    room = torch.empty(2 * k * n, device=DEV).view(k, 2, n)
    p = [room[k - 1 - i, i % 2] for i in range(k)]
    m = [room[k - 1 - i, 1 - i % 2] for i in range(k)]
    g = [values[0, i // 2] for i in range(k)]
    for x, y in zip(p, values[1]):
        x.copy_(y)
    own = [y.clone() for y in values[1]]
    zero = lambda: [torch.zeros(n, device=DEV) for _ in range(k)]  # noqa: E731
    if bits == 32:
        for x in m:
            x.zero_()
        mine, theirs = (m, zero(), None), (zero(), zero(), None)
    else:                                                # codes and scales in what the moments would take
        q = [x.view(torch.int8)[:n].view(4, 256).zero_() for x in m]
        c = [x.view(torch.uint8)[n:2 * n].view(4, 256).zero_() for x in m]
        s = [x[512:520].view(4, 2).zero_() for x in m]
        mine, theirs = (q, c, s), tuple(map(list, zip(*(optim.moments8_encode(x, x) for x in zero()))))
    hyper = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    for _ in range(2):
        run(p, g, *mine, torch.zeros(k, device=DEV), 0.5, **hyper)
        run(own, [x.clone() for x in g], *theirs, torch.zeros(k, device=DEV), 0.5, **hyper)
    assert all(torch.equal(x, y) for x, y in zip(p, own))
    assert all(torch.equal(x, y) for a, b in zip(mine, theirs) if a is not None for x, y in zip(a, b))


@pytest.mark.parametrize("device", ["cpu", DEV])
@pytest.mark.parametrize("eps", [1e-30, 1e-20, 1e-17, 1e-8])
@pytest.mark.parametrize("bits", [32, 8])
def test_second_moments_below_the_normal_numbers(bits, eps, device):
    """First steps of gradients from 3e-20 to 1e-15: v = 0.001 g^2 goes from 9e-43, where fp32 has steps of 2^-149, to
    1e-33.  Its one rounding to such a step is off by half of it, so a root by 2^-150 / (2 v) of itself (4e-4 at most)
    beside the usual; twice that is allowed, since the formula's root is taken at v as it was."""
    n = 3000
    gen = torch.Generator().manual_seed(6)
    g = torch.exp(torch.empty(n).uniform_(math.log(3e-20), math.log(1e-15), generator=gen)) * (torch.rand(n, generator=gen) - 0.5).sign()
    p = 0.05 * torch.randn(n, generator=gen)
    hyper = dict(lr=1e-3, betas=(0.9, 0.999), eps=eps, weight_decay=0.0)
    zero = torch.zeros(n)
    want, bound = U.step64(p, g, zero, zero, 1, **hyper)
    update = (want[0] - p.double()).abs()
    bound = bound[0] + update * 2.0 ** -149 / (2 * want[2].clamp(min=2.0 ** -149))
    m, v, s = (zero.clone(), zero.clone(), None) if bits == 32 else optim.moments8_encode(zero, zero)
    to = lambda x: [x.to(device)]  # noqa: E731
    here = to(p.clone())
    run(here, to(g), to(m), to(v), None if s is None else to(s), torch.zeros(1, device=device), None, **hyper)
    U.assert_near(here[0], want[0], bound, f"eps {eps}")


@pytest.mark.parametrize("device", ["cpu", DEV])
def test_small_second_moments_beside_large_ones_keep_a_code(device):
    """A v above zero has c >= 1 after a step too, however small it is: one element of each block has a gradient of 1."""
    g = torch.full((1024,), 1e-19)                       # 0.001 g^2 = 1e-41
    g[::256], g[5::256] = 1.0, 0.0
    zero = torch.zeros(1024)
    q, c, s = (x.to(device) for x in optim.moments8_encode(zero, zero))
    optim.adamw8_step([torch.ones(1024, device=device)], [g.to(device)], [q], [c], [s], torch.zeros(1, device=device), lr=1e-3)
    want = torch.ones(4, 256, dtype=torch.uint8)
    want[:, 0], want[:, 5] = 255, 0
    assert torch.equal(c.cpu(), want)


@pytest.mark.parametrize("bits", [(8, 8), (8, 32), (32, 8)])
@pytest.mark.parametrize("target", LAYOUTS)
@pytest.mark.parametrize("source", LAYOUTS)
def test_load_state_dict_into_another_order_of_memory(source, target, bits):
    check_load_of_another_order(source, target, bits, DEV)


def test_a_parameter_whose_order_changes_under_its_codes():
    opt, p = optimizer_of("contiguous", 8, DEV)
    p.data = p.data.contiguous(memory_format=torch.channels_last)
    p.grad = torch.ones_like(p)
    before = p.detach().clone()
    with pytest.raises(ValueError, match="order"):
        opt.step()
    assert torch.equal(p, before) and float(opt.state[p]["step"]) == 2
    opt, p = optimizer_of("contiguous", 8, DEV, shape=(8, 16, 1, 1))
    p.data = p.data.contiguous().as_strided(p.shape, (16, 1, 16, 16))
    p.grad = torch.ones_like(p)
    opt.step()
    assert float(opt.state[p]["step"]) == 3


@pytest.mark.parametrize("device", ["cpu", DEV])
def test_negated_views_are_taken_by_value(device):
    """A view that torch keeps as "the negative of this memory" (the imaginary part of a conjugate) is its values."""
    x = torch.randn(600, generator=torch.Generator().manual_seed(0)).to(device)
    neg = torch._neg_view(x)
    assert neg.is_neg() and torch.equal(neg, -x)
    for got, want in zip(optim.moments8_encode(neg, x.abs()), optim.moments8_encode(-x, x.abs())):
        assert torch.equal(got, want)
    for got, want in zip(optim.grad_norm([neg]), optim.grad_norm([x])):
        assert torch.equal(got, want)
    ends = []
    for g in (neg, -x):
        p = [torch.ones(600, device=device)]
        optim.adamw_step(p, [g], [torch.zeros(600, device=device)], [torch.zeros(600, device=device)], torch.zeros(1, device=device), lr=1e-2)
        ends.append(p[0])
    assert torch.equal(*ends)
