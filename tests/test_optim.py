"""pir_amd.optim on the CPU: the torch form against 64 bits, the refusals, the optimizer class, its checkpoints, and the
host checks of the C entry points (which come before any launch)."""
import ctypes
import math

import pytest
import torch

import optim_util as U
from pir_amd import optim, train

SIZES = [0, 1, 2, 255, 256, 257, 1000]


def run(p, g, m, v, s, steps, max_norm, **hyper):
    if s is None:
        return optim.adamw_step(p, g, m, v, steps, max_norm=max_norm, **hyper)
    return optim.adamw8_step(p, g, m, v, s, steps, max_norm=max_norm, **hyper)


@pytest.mark.parametrize("max_norm", [None, 1e-3, 10.0, math.inf])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", U.TYPES)
def test_torch_form_matches_64_bits(dtype, bits, max_norm):
    U.check_step(run, SIZES, dtype, bits, "cpu", odd=True, max_norm=max_norm)


def test_grad_norm_on_the_cpu():
    g = [torch.randn(n, generator=torch.Generator().manual_seed(n)) for n in (1, 7, 300)] + [torch.zeros(0)]
    total, each = optim.grad_norm(g)
    assert abs(float(total) - U.norm64(g)) <= 1.001 * U.E * U.norm64(g) and each.shape == (4,) and float(each[3]) == 0.0


def lists(n=300, bits=32, count=2):
    p, g, m, v, s, steps = U.make([n] * count, torch.float32, bits, "cpu")
    return dict(params=p, grads=g, exp_avgs=m, exp_avg_sqs=v, steps=steps, **({} if s is None else {"scales": s}))


@pytest.mark.parametrize("what, change", [
    ("a list too short", dict(grads=lambda x: x[:1])),
    ("one gradient missing", dict(grads=lambda x: [x[0], None])),
    ("a gradient of another type", dict(grads=lambda x: [x[0], x[1].half()])),
    ("a gradient of another shape", dict(grads=lambda x: [x[0], x[1][:-1]])),
    ("a sparse gradient", dict(grads=lambda x: [x[0], x[1].to_sparse()])),
    ("a parameter of another type", dict(params=lambda x: [x[0], x[1].double()], grads=lambda x: [x[0], x[1].double()])),
    ("a parameter with gaps", dict(params=lambda x: [x[0], torch.zeros(600)[::2]])),
    ("a parameter that is one element, expanded", dict(params=lambda x: [x[0], torch.zeros(1).expand(300)])),
    ("a parameter twice", dict(params=lambda x: [x[0], x[0]])),
    ("parameters that overlap", dict(params=lambda x: (lambda b: [b[:300], b[299:599]])(torch.zeros(599)))),
    ("one list for both moments", dict(exp_avg_sqs=lambda x: "exp_avgs")),
    ("the parameters for a moment", dict(exp_avgs=lambda x: "params")),
    ("a moment twice", dict(exp_avgs=lambda x: [x[1], x[1]])),
    ("a moment of another type", dict(exp_avg_sqs=lambda x: [x[0], x[1].bfloat16()])),
    ("a moment of another shape", dict(exp_avgs=lambda x: [x[0], x[1].view(30, 10)])),
    ("step counts of another type", dict(steps=lambda x: x.int())),
    ("a step count too few", dict(steps=lambda x: x[:1])),
    ("a step count of each kind, strided", dict(steps=lambda x: torch.zeros(4)[::2])),
    ("lr below zero", dict(lr=-1.0)), ("lr not a number", dict(lr=math.nan)), ("lr of two", dict(lr=torch.ones(2))),
    ("beta1 of one", dict(betas=(1.0, 0.9))), ("beta2 below zero", dict(betas=(0.9, -0.1))),
    ("eps below zero", dict(eps=-1e-8)), ("decay below zero", dict(weight_decay=-1.0)), ("decay infinite", dict(weight_decay=math.inf)),
    ("max_norm of zero", dict(max_norm=0.0)), ("max_norm not a number", dict(max_norm=math.nan)),
])
def test_step_refuses(what, change):
    args = dict(lists(), lr=1e-3)
    before = {k: [t.clone() for t in args[k]] for k in ("params", "exp_avgs", "exp_avg_sqs")}
    for k, f in change.items():
        args[k] = f(args[k]) if callable(f) and k not in ("lr",) else f
        args[k] = args[args[k]] if isinstance(args[k], str) else args[k]
    lists_only = {k: args.pop(k) for k in ("params", "grads", "exp_avgs", "exp_avg_sqs", "steps")}
    kept = lists(), before
    with pytest.raises(ValueError):
        optim.adamw_step(*lists_only.values(), **args)
    assert all(torch.equal(a, b) for k in before for a, b in zip(kept[0][k], before[k])), what


@pytest.mark.parametrize("what, change", [
    ("codes of the wrong count", dict(exp_avgs=lambda x: [x[0], x[1][:1]])),
    ("codes of the wrong type", dict(exp_avgs=lambda x: [x[0], x[1].view(torch.uint8)])),
    ("scales of the wrong shape", dict(scales=lambda x: [x[0], x[1][:, :1]])),
    ("scales of the wrong type", dict(scales=lambda x: [x[0], x[1].double()])),
    ("scales too few", dict(scales=lambda x: x[:1])),
    ("codes off their alignment", dict(exp_avgs=lambda x: [x[0], torch.zeros(513, dtype=torch.int8)[1:].view(2, 256)])),
    ("eps below what the 8-bit step resolves", dict(eps=1e-31)),
    ("codes with gaps", dict(exp_avg_sqs=lambda x: [x[0], torch.zeros(2, 512, dtype=torch.uint8)[:, ::2]])),
])
def test_8_bit_step_refuses(what, change):
    args = dict(lists(bits=8), eps=1e-8)
    for k, f in change.items():
        args[k] = f(args[k]) if callable(f) else f
    with pytest.raises(ValueError):
        optim.adamw8_step(*(args[k] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs", "scales", "steps")), lr=1e-3,
                          eps=args["eps"])


def test_no_parameters_is_no_work():
    assert optim.adamw_step([], [], [], [], torch.zeros(0), lr=1e-3) is None
    assert float(optim.adamw_step([], [], [], [], torch.zeros(0), lr=1e-3, max_norm=1.0)) == 0.0
    with pytest.raises(ValueError):
        optim.grad_norm([])


def test_norm_and_moments_refuse():
    with pytest.raises(ValueError):
        optim.grad_norm([torch.zeros(3, dtype=torch.float64)])
    with pytest.raises(ValueError):
        optim.grad_norm([torch.zeros(3).to_sparse()])
    q, c, s = optim.moments8_encode(torch.randn(300), torch.rand(300))
    for bad in ((q.view(-1), c, s), (q, c[:1], s), (q, c, s[:, :1]), (c, q, s), (q, c, s.double())):
        with pytest.raises(ValueError):
            optim.moments8_decode(*bad)
    with pytest.raises(ValueError):
        optim.moments8_decode(q, c, s, dtype=torch.float64)
    for bad in ((torch.zeros(3), torch.zeros(4)), (torch.zeros(3), torch.zeros(3).half()),
                (torch.zeros(3, dtype=torch.float64),) * 2, (torch.zeros(6)[::2],) * 2):
        with pytest.raises(ValueError):
            optim.moments8_encode(*bad)


def test_moments8_round_trip():
    """Half a step of the nearest code: of m = a x^2 with x in steps of 1/127 that is at most a (x + 1/254) / 127 with the
    rounding's own square (1/254)^2 a; of v = b x^4 the same with 255 and its derivative."""
    gen = torch.Generator().manual_seed(1)
    m = torch.randn(10_000, generator=gen) * torch.exp(3 * torch.randn(10_000, generator=gen))
    v = m ** 2 * torch.rand(10_000, generator=gen)
    q, c, s = optim.moments8_encode(m, v)
    U.assert_coded(q, c, s, m.double(), v.double(), 2 * U.E * m.double().abs(), 2 * U.E * v.double(), "encode")
    a, b = (x.reshape(-1)[:10_000] for x in optim.moments8_decode(q, c, s))
    top = s.repeat_interleave(256, 0)[:10_000]
    x = (m.abs() / top[:, 0]).sqrt()
    assert bool(((a - m).abs() <= top[:, 0] * ((x + 1 / 254) / 127 + 1 / 254 ** 2) + 1e-6 * m.abs()).all())
    assert bool((b[v > 0] > 0).all())                  # no second moment is lost
    y = (v / top[:, 1]) ** 0.25
    half = torch.where(y > 1 / 255, 0.5 / 255, 1 / 255)
    assert bool(((b - v).abs() <= top[:, 1] * ((y + half) ** 4 - (y - half).clamp(min=0) ** 4) + 1e-6 * v).all())


def test_moments8_special_blocks():
    m, v = torch.ones(6 * 256), torch.ones(6 * 256)
    m[:256], v[:256] = 0.0, 0.0                         # nothing there
    m[256:512] = 1e-39                                  # below 2^-126
    m[512 + 7], v[768 + 9], m[1024] = math.inf, math.nan, -math.inf
    q, c, s = optim.moments8_encode(m, v)
    a, b = optim.moments8_decode(q, c, s)
    assert float(a[0].abs().max()) == 0 and float(b[0].max()) == 0 and float(a[1].abs().max()) == 0 and bool((b[1] == 1).all())
    assert bool(a[2].isnan().all()) and bool((b[2] == 1).all()) and bool(b[3].isnan().all()) and bool(a[4].isnan().all())
    assert bool((a[5] == 1).all()) and bool((b[5] == 1).all())


def networks(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(3, 80), torch.nn.ReLU(), torch.nn.Linear(80, 90), torch.nn.ReLU(), torch.nn.Linear(90, 1))


def train_steps(net, opt, steps, seed=0):
    gen = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        opt.zero_grad()
        x = torch.randn(32, 3, generator=gen)
        ((net(x) - x.sum(1, keepdim=True)) ** 2).mean().backward()
        opt.step()


def assert_moved_alike(a, b, start, lr, steps, part=1e-3):
    """Parameters after the same steps: an fp32 step of Adam is at most about lr long and two evaluations of it agree to a
    few 1e-5 of it, unless the gradient is rounding noise."""
    for x, y, z in zip(a.parameters(), b.parameters(), start):
        off = (x - y).abs() / lr
        assert float(off.quantile(0.99)) <= part * steps, float(off.max())
        assert not torch.equal(x, z)


@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_class_takes_the_steps_of_torch(decay):
    ours, theirs = networks(), networks()
    start = [p.detach().clone() for p in ours.parameters()]
    a = optim.AdamW(ours.parameters(), lr=1e-3, weight_decay=decay)
    b = torch.optim.AdamW(theirs.parameters(), lr=1e-3, weight_decay=decay)
    train_steps(ours, a, 6)
    train_steps(theirs, b, 6)
    assert_moved_alike(ours, theirs, start, 1e-3, 6)


def test_class_state_and_skipped_parameters():
    net = networks()
    opt = optim.AdamW(net.parameters(), state_bits=8)
    list(net.parameters())[0].grad = None
    opt.step()
    assert len(opt.state) == 0                           # no gradients: no state, no step counted
    ps = list(net.parameters())
    for p in ps[1:]:
        p.grad = torch.ones_like(p)
    opt.step()
    assert ps[0] not in opt.state and len(opt.state) == len(ps) - 1 and float(opt.state[ps[1]]["step"]) == 1
    assert opt.state[ps[2]]["exp_avg"].dtype == torch.int8 and opt.state[ps[2]]["scales"].shape == (29, 2)   # 80 x 90
    assert opt.state[ps[1]]["exp_avg"].dtype == torch.float32 and "scales" not in opt.state[ps[1]]
    assert opt.total_norm is None
    opt.max_norm = 1.0
    opt.step()
    assert abs(float(opt.total_norm) - math.sqrt(sum(p.numel() for p in ps[1:]))) < 1e-4


@pytest.mark.parametrize("kw", [dict(lr=-1), dict(betas=(0.9, 1.0)), dict(eps=-1), dict(weight_decay=-1), dict(state_bits=16),
                                dict(max_norm=-1.0)])
def test_class_refuses(kw):
    with pytest.raises(ValueError):
        optim.AdamW(networks().parameters(), **kw)


def test_step_together_is_the_steps_with_one_norm():
    nets = [networks(1), networks(2)]
    copies = [networks(1), networks(2)]
    for pair in (nets, copies):
        for net in pair:
            net(torch.randn(32, 3, generator=torch.Generator().manual_seed(3))).pow(2).mean().backward()
    opts = [optim.AdamW(net.parameters(), lr=lr, state_bits=bits) for net, lr, bits in zip(nets, (1e-3, 1e-4), (32, 8))]
    norm = optim.step_together(opts, max_norm=0.01)
    total = torch.nn.utils.clip_grad_norm_([p for net in copies for p in net.parameters()], 0.01)
    assert abs(float(norm) - float(total)) < 1e-6 * float(total)
    for net, copy, lr, bits in zip(nets, copies, (1e-3, 1e-4), (32, 8)):
        optim.AdamW(copy.parameters(), lr=lr, state_bits=bits).step()
        for x, y in zip(net.parameters(), copy.parameters()):
            assert float((x - y).abs().max()) <= 1e-3 * lr
    with pytest.raises(ValueError):
        optim.step_together([opts[0], opts[0]])
    with pytest.raises(TypeError):
        optim.step_together([torch.optim.Adam(nets[0].parameters())])
    assert float(optim.step_together([], max_norm=1.0)) == 0.0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("source", ["torch", 32, 8])
def test_load_state_dict(source, bits):
    """A run continues from the state of this class or of torch.optim.Adam as it would have without the break: to the bit in
    32 bits and from 8 to 8, to the moments' rounding otherwise."""
    net, other = networks(), networks()
    make = lambda n, b: torch.optim.Adam(n.parameters(), lr=1e-3) if b == "torch" else \
        optim.AdamW(n.parameters(), lr=1e-3, weight_decay=0.0, state_bits=b, min_8bit_numel=100)  # noqa: E731
    first = make(net, source)
    train_steps(net, first, 4)
    other.load_state_dict(net.state_dict())
    second = make(other, bits)
    second.load_state_dict(first.state_dict())
    assert second.param_groups[0]["lr"] == 1e-3
    second.param_groups[0]["state_bits"] = bits
    second.load_state_dict({**first.state_dict(), "param_groups": [{**first.state_dict()["param_groups"][0], "state_bits": bits}]})
    start = [p.detach().clone() for p in net.parameters()]
    train_steps(net, first, 1, seed=9)
    train_steps(other, second, 1, seed=9)
    for p in other.parameters():
        assert float(second.state[p]["step"]) == 5
        assert ("scales" in second.state[p]) == (bits == 8 and p.numel() >= 100)
    # moments rounded to 8 bits move a step by some percent of its length
    assert_moved_alike(net, other, start, 1e-3, 1, part=1e-3 if source != 8 and bits == 32 or source == bits else 0.3)
    back = torch.optim.AdamW(networks().parameters(), lr=1e-3)
    if bits == 32:
        back.load_state_dict(second.state_dict())        # and torch takes it back
        assert float(list(back.state.values())[0]["step"]) == 5


def test_copies_of_the_optimizer_keep_its_settings():
    import copy
    net = networks()
    opt = copy.deepcopy(optim.AdamW(net.parameters(), max_norm=0.5, skip_nonfinite=True, state_bits=8))
    for g in opt.param_groups:
        for p in g["params"]:
            p.grad = torch.ones_like(p)
    opt.step()
    assert opt.max_norm == 0.5 and opt.skip_nonfinite and float(opt.total_norm) > 1 and opt.param_groups[0]["state_bits"] == 8


def test_load_state_dict_refuses():
    net = networks()
    opt = optim.AdamW(net.parameters())
    for bad in (torch.optim.Adam(net.parameters(), amsgrad=True), torch.optim.Adam(net.parameters(), weight_decay=0.1),
                torch.optim.AdamW(net.parameters(), maximize=True)):
        with pytest.raises(ValueError):
            opt.load_state_dict(bad.state_dict())


def test_load_state_dict_refuses_other_shapes():
    net = networks()
    opt = optim.AdamW(net.parameters())
    train_steps(net, opt, 1)
    saved = opt.state_dict()
    saved["state"][0] = {**saved["state"][0], "exp_avg": torch.zeros(1)}
    with pytest.raises(ValueError):
        optim.AdamW(networks().parameters()).load_state_dict(saved)


def test_skip_nonfinite_changes_nothing():
    p, g, m, v, _, steps = U.make([300, 5], torch.float32, 32, "cpu")
    keep = [t.clone() for x in (p, m, v) for t in x]
    g[1][2] = math.inf
    norm = optim.adamw_step(p, g, m, v, steps, lr=1e-3, max_norm=1.0, skip_nonfinite=True)
    assert float(norm) == math.inf and steps.tolist() == [3.0, 4.0]
    assert all(torch.equal(a, b) for a, b in zip(keep, [t for x in (p, m, v) for t in x]))


def test_step_optimizers_of_a_training_run():
    nets = {k: networks(i) for i, k in enumerate(("diffuse_albedo_network", "specular_albedo_network"))}

    class Light(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.light, self.light_offset = torch.nn.Parameter(torch.tensor(1.0)), torch.nn.Linear(3, 1, bias=False)
    nets["point_light_network"] = Light()
    lr = {"sdf_network": 1e-5, "diffuse_albedo_network": 1e-4, "specular_albedo_network": 1e-4}
    for kind in ("adam", "adamw", "adamw8"):
        sdf = networks(7)
        sdf_opt, color, dino = train.make_optimizers(sdf, nets, networks(8), lr, True, optimizer=kind)
        assert isinstance(sdf_opt, torch.optim.Adam if kind == "adam" else optim.AdamW)
        assert [g["lr"] for g in color["point_light_network"].param_groups] == [2e-5, 1e-4]
        for p in sdf.parameters():
            p.grad = torch.ones_like(p)
        norm = train.step_optimizers([sdf_opt, color["point_light_network"]], 0.5)
        assert abs(float(norm) - math.sqrt(sum(p.numel() for p in sdf.parameters()))) < 1e-3
        assert train.step_optimizers([sdf_opt]) is None
    with pytest.raises(ValueError):
        train.make_optimizers(networks(7), nets, networks(8), lr, True, optimizer="sgd")


def test_training_steps_with_adamw(monkeypatch):
    """Two iterations of the training loop with torch.optim.Adam and with this package's AdamW: the parameters they step
    end at the same place, to a few 1e-5 of a step of lr where the gradient is no rounding noise."""
    import functools
    import numpy as np
    import train_traj_util
    make = train.make_optimizers
    ends = []
    for kind in ("adam", "adamw"):
        monkeypatch.setattr(train, "make_optimizers", functools.partial(make, optimizer=kind))
        d, state = train_traj_util.build_state("cpu")
        np.random.seed(int(d["np_seed"]))
        start = [p.detach().clone() for p in state.sdf_network.parameters()]
        for i in range(2):
            train.training_step(state, int(d["first_step"]) + i, eik_points=torch.from_numpy(d["eik_points"][i]))
        ends.append(list(state.sdf_network.parameters()))
    moved = 0
    for x, y, z in zip(*ends, start):
        if x.numel() >= 256 and not torch.equal(x, z):
            moved += 1
            assert float(((x - y).detach().abs() / 1e-5).quantile(0.95)) < 0.05
    assert moved > 10


# ---- the C entry points' host checks: every call here is refused before anything is launched
class Group(ctypes.Structure):
    _fields_ = [(k, ctypes.c_double) for k in ("lr", "beta1", "beta2", "eps", "weight_decay")] + [("lr_device", ctypes.c_void_p)]


def c_step(n=1, **change):
    from pir_amd import _lib
    L = _lib.lib()
    one = (ctypes.c_void_p * 4)(*[4096] * 4)             # never read: the checks come first
    args = dict(params=one, grads=one, m=one, v=one, scales=None, steps=one, numels=(ctypes.c_long * 4)(*[10] * 4),
                dtypes=(ctypes.c_int * 4)(), groups=(ctypes.c_int * 4)(), group=(Group * 1)(Group(1e-3, 0.9, 0.99, 1e-8, 0.0, None)),
                n_groups=1, max_norm=0.0, skip=0, norm=None, work=4096, size=0, stream=None)
    args.update(change)
    at = lambda x: ctypes.addressof(x) if isinstance(x, ctypes.Array) else x  # noqa: E731
    return L.pir_adamw_step(n, *[at(x) for x in args.values()])


@pytest.mark.parametrize("code, change", [
    (1, dict(n=-1)), (1, dict(params=None)), (1, dict(grads=None)), (1, dict(m=None)), (1, dict(steps=None)), (1, dict(numels=None)),
    (1, dict(groups=None)), (1, dict(group=None)), (1, dict(n_groups=0)),
    (1, dict(numels=(ctypes.c_long * 1)(-1))), (1, dict(dtypes=(ctypes.c_int * 1)(3))), (1, dict(groups=(ctypes.c_int * 1)(1))),
    (1, dict(grads=(ctypes.c_void_p * 1)(None))), (1, dict(params=(ctypes.c_void_p * 1)(None))), (1, dict(steps=(ctypes.c_void_p * 1)(None))),
    (1, dict(scales=(ctypes.c_void_p * 1)(4), m=(ctypes.c_void_p * 1)(4096))),
    (1, dict(scales=(ctypes.c_void_p * 1)(4096), m=(ctypes.c_void_p * 1)(4100))),
    (1, dict(group=(Group * 1)(Group(1e-3, 1.0, 0.99, 1e-8, 0.0, None)))),
    (1, dict(group=(Group * 1)(Group(math.nan, 0.9, 0.99, 1e-8, 0.0, None)))),
    (1, dict(params=(ctypes.c_void_p * 1)(4098))), (1, dict(steps=(ctypes.c_void_p * 1)(4097))),
    (1, dict(scales=(ctypes.c_void_p * 1)(4096), group=(Group * 1)(Group(1e-3, 0.9, 0.99, 1e-31, 0.0, None)))),
    (3, dict(size=16)), (3, dict(work=None, size=1 << 20)),
    (4, dict(numels=(ctypes.c_long * 1)(1 << 60))),
])
def test_c_step_refuses(code, change):
    assert c_step(**change) == code


def test_c_calls_without_work():
    from pir_amd import _lib
    L = _lib.lib()
    assert c_step(n=0) == 0
    assert L.pir_adamw_workspace_bytes(-1, None, 0) == 0 and L.pir_grad_norm_workspace_bytes(2, None) == 0
    assert L.pir_moments8_decode(0, None, None, None, 0, None, None, None) == 0
    assert L.pir_moments8_decode(1, None, None, None, 0, None, None, None) == 1
    assert L.pir_moments8_decode(-1, None, None, None, 0, None, None, None) == 1
    assert L.pir_moments8_encode(0, 0, None, None, None, None, None, None) == 0
    assert L.pir_moments8_encode(5, 7, None, None, None, None, None, None) == 1
    assert L.pir_grad_norm(1, None, None, None, None, None, None, 0, None) == 1


class Elsewhere(torch.nn.Parameter):
    """A parameter that says it lives on another device."""

    def get_device(self):
        return 7


@pytest.mark.parametrize("ask", [dict(max_norm=1.0), dict(max_norm=math.inf), dict(skip_nonfinite=True)])
def test_a_joint_norm_over_devices_is_refused(ask):
    """Whatever it is for, clipping, skipping or being looked at; and before anything has a state."""
    ps = [torch.nn.Parameter(torch.ones(9)), Elsewhere(torch.ones(16))]
    for p in ps:
        p.grad = torch.ones(p.shape)
    opt = optim.AdamW(ps, **ask)
    with pytest.raises(ValueError, match="several devices"):
        opt.step()
    with pytest.raises(ValueError, match="several devices"):
        optim.step_together([opt], **ask)
    assert len(opt.state) == 0 and all(torch.equal(p, torch.ones(p.shape)) for p in ps)
    assert optim.step_together([opt]) is None and all(float(opt.state[p]["step"]) == 1 for p in ps)


def overlaps(bits):
    """What one call may not be given: two of the tensors it writes, or one of those and a gradient, share memory."""
    cases = {
        "moments crossed": lambda a: a.update(exp_avg_sqs=a["exp_avgs"][::-1]) if bits == 32 else
        a.update(exp_avg_sqs=[t.view(torch.uint8) for t in a["exp_avgs"][::-1]]),
        "a step count twice": lambda a: a.update(steps=[a["steps"][:1].view(()), a["steps"][:1].view(())]),
        "step counts in a parameter": lambda a: a.update(steps=a["params"][1][10:12]),
        "a gradient that is a parameter": lambda a: a.update(grads=a["params"]),
        "a gradient that starts inside a parameter": lambda a: a.update(grads=[a["grads"][0], a["room"][100:400]],
                                                                        params=[a["params"][0], a["room"][:300]]),
    }
    if bits == 32:
        cases["a parameter that ends inside a moment"] = lambda a: a.update(params=[a["params"][0], a["room"][:300]],
                                                                            exp_avgs=[a["room"][299:599], a["exp_avgs"][1]])
        cases["a gradient that is another's moment"] = lambda a: a.update(grads=[a["exp_avg_sqs"][1], a["grads"][1]])
    else:
        cases["scales twice"] = lambda a: a.update(scales=[a["scales"][0]] * 2)
        cases["scales that overlap"] = lambda a: a.update(scales=[a["room"][:4].view(2, 2), a["room"][2:6].view(2, 2)])
        cases["scales in a parameter"] = lambda a: a.update(scales=[a["scales"][0], a["params"][0][100:104].view(2, 2)])
    return cases


def refused_call(bits, what, device="cpu"):
    """Makes one of those calls, through the list call or, for lists of step counts, as the class makes it; nothing of what
    it was given may have moved."""
    args = {k: [t.to(device) for t in v] if isinstance(v, list) else v.to(device) for k, v in lists(bits=bits).items()}
    args["room"] = torch.zeros(600, device=device)
    overlaps(bits)[what](args)
    del args["room"]
    given = [t for v in args.values() for t in v]        # the very tensors of the call, its step counts among them
    before = [t.clone() for t in given]
    with pytest.raises(ValueError, match="overlap"):
        if isinstance(args["steps"], list):
            from array import array
            run_list = optim._run if device == "cuda" else optim._run_torch
            grads = args["grads"] if device == "cuda" else optim._check(*(args.get(k) for k in (
                "params", "grads", "exp_avgs", "exp_avg_sqs", "scales", "steps")))
            run_list(args["params"], grads, args["exp_avgs"], args["exp_avg_sqs"], args.get("scales"), args["steps"],
                     array("i", [0, 0]), [(1e-3, 0.9, 0.999, 1e-8, 0.0, 0)], 0.0, False, False)
        else:
            (optim.adamw8_step if bits == 8 else optim.adamw_step)(*[args[k] for k in (
                "params", "grads", "exp_avgs", "exp_avg_sqs", "scales", "steps") if k in args], lr=1e-3)
    assert all(torch.equal(a, b) for a, b in zip(given, before))


@pytest.mark.parametrize("bits, what", [(b, w) for b in (32, 8) for w in overlaps(b)])
def test_overlapping_tensors_are_refused(bits, what):
    refused_call(bits, what)


def test_one_gradient_for_two_parameters():
    """Gradients are only read: they may share memory."""
    g = torch.randn(300, generator=torch.Generator().manual_seed(0))
    p = [torch.ones(300), torch.ones(300)]
    m, v = ([torch.zeros(300), torch.zeros(300)] for _ in "mv")
    optim.adamw_step(p, [g, g], m, v, torch.zeros(2), lr=1e-3)
    assert torch.equal(p[0], p[1]) and torch.equal(m[0], m[1]) and not torch.equal(p[0], torch.ones(300))


def assert_same_moments(a, pa, b, pb, parts):
    """Moments of two optimizers' parameters: alike to the bit, or to parts (first, second) of their block's largest."""
    def values(opt, p):
        s = opt.state[p]
        if "scales" not in s:
            return s["exp_avg"], s["exp_avg_sq"]
        flat = [x.reshape(-1)[:p.numel()] for x in optim.moments8_decode(s["exp_avg"], s["exp_avg_sq"], s["scales"])]
        return [x.as_strided(p.shape, p.stride()) for x in flat]
    for x, y, part in zip(values(a, pa), values(b, pb), parts):
        assert float((x - y).abs().max()) <= part * float(x.abs().max())


# the largest error of a code: at x = 1 of x^2 in steps of 1/127, and of x^4 in steps of 1/255 (the least code stands for
# more than that only below 2.5e-10), with the rounding's own square and the fp32 evaluation
CODE_PARTS = (1 / 127 + 1 / 254 ** 2, 2 / 255 + 6 * (0.5 / 255) ** 2 + 1e-6)


@pytest.mark.parametrize("source", ["torch", 32, 8])
def test_load_state_dict_keeps_the_optimizers_own_bits(source):
    """Whatever the state comes from, each group holds it in its own number of bits, and takes the other settings."""
    net, other = networks(), networks()
    ours = lambda n, **k: optim.AdamW(n.parameters(), lr=3e-3, weight_decay=0.0, **k)  # noqa: E731
    first = torch.optim.Adam(net.parameters(), lr=3e-3) if source == "torch" else ours(net, state_bits=source, min_8bit_numel=50)
    train_steps(net, first, 3)
    for bits, least in ((32, 4096), (8, 4096), (8, 100)):
        second = optim.AdamW(other.parameters(), lr=1e-4, state_bits=bits, min_8bit_numel=least)
        second.load_state_dict(first.state_dict())
        g = second.param_groups[0]
        assert (g["state_bits"], g["min_8bit_numel"], g["lr"], g["weight_decay"]) == (bits, least, 3e-3, 0.0)
        for p, q in zip(net.parameters(), other.parameters()):
            coded = bits == 8 and q.numel() >= least
            assert ("scales" in second.state[q]) == coded and float(second.state[q]["step"]) == 3
            moved = coded != ("scales" in first.state[p])
            assert_same_moments(first, p, second, q, CODE_PARTS if moved else (0.0, 0.0))


@pytest.mark.parametrize("source", ["torch", 32])
def test_load_state_dict_into_groups_of_their_own(source):
    net = networks()
    halves = lambda: [{"params": list(net.parameters())[:3]}, {"params": list(net.parameters())[3:]}]  # noqa: E731
    first = torch.optim.AdamW(halves(), lr=1e-3) if source == "torch" else optim.AdamW(halves(), lr=1e-3)
    train_steps(net, first, 2)
    second = optim.AdamW([{**halves()[0], "state_bits": 8, "min_8bit_numel": 1}, halves()[1]], lr=1e-4)
    second.load_state_dict(first.state_dict())
    assert [g["state_bits"] for g in second.param_groups] == [8, 32] and [g["lr"] for g in second.param_groups] == [1e-3, 1e-3]
    assert ["scales" in second.state[p] for p in net.parameters()] == [True] * 3 + [False] * 3


@pytest.mark.parametrize("gone", ["step", "exp_avg", "exp_avg_sq"])
@pytest.mark.parametrize("source", ["torch", 32, 8])
def test_load_state_dict_refuses_a_state_with_a_part_missing(source, gone):
    net = networks()
    first = torch.optim.Adam(net.parameters()) if source == "torch" else optim.AdamW(net.parameters(), state_bits=source, min_8bit_numel=1)
    train_steps(net, first, 1)
    saved = first.state_dict()
    saved["state"][2] = {k: v for k, v in saved["state"][2].items() if k != gone}
    for bits in (32, 8):
        with pytest.raises(ValueError, match=f"parameter 2.*{gone}"):
            optim.AdamW(networks().parameters(), state_bits=bits, min_8bit_numel=1).load_state_dict(saved)


def test_load_state_dict_refuses_codes_of_another_type():
    """Codes that a cast made numbers of another type are no codes."""
    net = networks()
    first = optim.AdamW(net.parameters(), state_bits=8, min_8bit_numel=1)
    train_steps(net, first, 1)
    for k, t in (("exp_avg", torch.float32), ("exp_avg_sq", torch.int8), ("scales", torch.bfloat16)):
        saved = first.state_dict()
        saved["state"][2] = {**saved["state"][2], k: saved["state"][2][k].to(t)}
        for bits in (32, 8):
            with pytest.raises(ValueError, match="parameter 2"):
                optim.AdamW(networks().parameters(), state_bits=bits, min_8bit_numel=1).load_state_dict(saved)


@pytest.mark.parametrize("bits", [32, 8])
def test_load_state_dict_that_fails_changes_nothing(bits):
    net, other = networks(), networks(3)
    first = optim.AdamW(net.parameters(), lr=5e-3)
    train_steps(net, first, 2)
    second = optim.AdamW(other.parameters(), lr=1e-3, state_bits=bits, min_8bit_numel=100)
    train_steps(other, second, 1)
    before = [(p, k, x, x.clone() if torch.is_tensor(x) else x) for p, s in second.state.items() for k, x in s.items()]
    for change in (lambda d: d["state"].update({5: {**d["state"][5], "exp_avg_sq": torch.zeros(2)}}),
                   lambda d: d["state"].update({5: {"step": torch.tensor(1.0)}}),
                   lambda d: d["param_groups"][0].update(amsgrad=True),
                   lambda d: d["param_groups"][0]["params"].pop()):
        saved = first.state_dict()
        change(saved)
        with pytest.raises(ValueError):
            second.load_state_dict(saved)
        assert second.param_groups[0]["lr"] == 1e-3 and len(second.state) == 6
        for p, k, x, y in before:
            now = second.state[p][k]
            assert now is x and (torch.equal(x, y) if torch.is_tensor(x) else x == y)


def test_load_state_dict_hooks_see_the_states():
    """Hooks before the load may put another state in place; hooks after it find the loaded one."""
    net = networks()
    first = optim.AdamW(net.parameters(), lr=1e-3)
    train_steps(net, first, 2)
    second = optim.AdamW(networks().parameters(), state_bits=8, min_8bit_numel=100)
    seen = []

    def before(opt, d):
        return {**d, "state": {k: {**s, "step": s["step"] + 40} for k, s in d["state"].items()}}

    def after(opt):
        seen.append([(float(opt.state[p]["step"]), "scales" in opt.state[p], opt.param_groups[0]["state_bits"])
                     for p in opt.param_groups[0]["params"]])
    second.register_load_state_dict_pre_hook(before)
    second.register_load_state_dict_post_hook(after)
    second.load_state_dict(first.state_dict())
    assert seen == [[(42.0, p.numel() >= 100, 8) for p in net.parameters()]]
    second.load_state_dict(first.state_dict())           # nothing of the load stays behind
    assert len(seen) == 2 and len(second._optimizer_load_state_dict_pre_hooks) == len(second._optimizer_load_state_dict_post_hooks) == 1


LAYOUTS = {
    "contiguous": lambda x: x.contiguous(),
    "channels_last": lambda x: x.contiguous(memory_format=torch.channels_last),
    "transposed": lambda x: x.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0),
}


def optimizer_of(layout, bits, device="cpu", steps=2, shape=(8, 16, 6, 6)):
    """An optimizer of one parameter whose memory is in some order, after some steps."""
    gen = torch.Generator().manual_seed(1)
    p = torch.nn.Parameter(LAYOUTS[layout](torch.randn(shape, generator=gen)).to(device))
    opt = optim.AdamW([p], lr=1e-3, state_bits=bits, min_8bit_numel=1)
    for _ in range(steps):
        p.grad = LAYOUTS[layout](torch.randn(shape, generator=gen) * torch.exp(torch.randn(shape, generator=gen))).to(device)
        opt.step()
    return opt, p


def check_load_of_another_order(source, target, bits, device):
    a, pa = optimizer_of(source, bits[0], device)
    b, pb = optimizer_of(target, bits[1], device, steps=0)
    assert pa.stride() == LAYOUTS[source](pa).stride() and pb.stride() == LAYOUTS[target](pb).stride()
    b.load_state_dict(a.state_dict())
    # in another order other elements share a scale, so codes are rounded once more: to the nearest of the new block's
    parts = CODE_PARTS if bits[1] == 8 and (bits[0] == 32 or source != target) else (1e-6, 1e-6) if bits[0] != bits[1] else (0.0, 0.0)
    assert_same_moments(a, pa, b, pb, parts)


@pytest.mark.parametrize("bits", [(8, 8), (8, 32), (32, 8), (32, 32)])
@pytest.mark.parametrize("target", LAYOUTS)
@pytest.mark.parametrize("source", LAYOUTS)
def test_load_state_dict_into_another_order_of_memory(source, target, bits):
    check_load_of_another_order(source, target, bits, "cpu")


def test_codes_without_a_record_of_their_order():
    """They are of a contiguous parameter: another cannot take them."""
    a, _ = optimizer_of("contiguous", 8)
    saved = a.state_dict()
    del saved["state"][0]["strides"]
    b, _ = optimizer_of("contiguous", 8, steps=0)
    b.load_state_dict(saved)
    for bits in (8, 32):
        c, _ = optimizer_of("channels_last", bits, steps=0)
        with pytest.raises(ValueError, match="order"):
            c.load_state_dict(saved)
    for bad in ((1, 1, 1, 1), (576, 36, 6, 2), (576, 36, 6), None, (-576, 36, 6, 1)):
        with pytest.raises(ValueError, match="order"):
            b.load_state_dict({**saved, "state": {0: {**saved["state"][0], "strides": bad}}})


def test_a_parameter_whose_order_changes_under_its_codes():
    """module.to(memory_format=...) moves a parameter's elements; codes cannot follow, and the step says so."""
    opt, p = optimizer_of("contiguous", 8)
    p.data = p.data.contiguous(memory_format=torch.channels_last)
    p.grad = torch.ones_like(p)
    before = p.detach().clone()
    with pytest.raises(ValueError, match="order"):
        opt.step()
    assert torch.equal(p, before)
    # strides of dimensions of one element say nothing
    opt, p = optimizer_of("contiguous", 8, shape=(8, 16, 1, 1))
    p.data = p.data.contiguous().as_strided(p.shape, (16, 1, 16, 16))
    p.grad = torch.ones_like(p)
    opt.step()
    assert float(opt.state[p]["step"]) == 3


@pytest.mark.parametrize("code, change", [
    (3, dict(work=4104, size=1 << 20)), (3, dict(work=4097, size=1 << 20)),     # descriptors are read from it 16 bytes at a time
    (1, dict(norm=4098, size=1 << 20)), (1, dict(group=(Group * 1)(Group(1e-3, 0.9, 0.99, 1e-8, 0.0, 4097)), size=1 << 20)),
])
def test_c_step_refuses_what_is_not_aligned(code, change):
    assert c_step(**change) == code


def test_c_calls_refuse_what_is_not_aligned():
    from pir_amd import _lib
    L = _lib.lib()
    one, numels, f32 = (ctypes.c_void_p * 1)(4096), (ctypes.c_long * 1)(10), (ctypes.c_int * 1)(0)
    at = [ctypes.addressof(x) for x in (one, numels, f32)]
    for total, each, work, code in ((4098, None, 4096, 1), (4096, 4097, 4096, 1), (4096, None, 4100, 3)):
        assert L.pir_grad_norm(1, *at, total, each, work, 1 << 16, None) == code
    for dtype, bad in ((0, 4098), (1, 4097), (2, 4097)):
        for m, v in ((bad, 4096), (4096, bad)):
            assert L.pir_moments8_decode(1, 4096, 4096, 4096, dtype, m, v, None) == 1
            assert L.pir_moments8_encode(5, dtype, m, v, 4096, 4096, 4096, None) == 1


@pytest.mark.parametrize("bad", [[None], [torch.ones(3), None], [torch.ones(3), 2.0]])
def test_grad_norm_refuses_what_is_no_tensor(bad):
    """A parameter without a gradient, above all: leaving it out is the caller's."""
    with pytest.raises(ValueError, match=f"tensor {len(bad) - 1}"):
        optim.grad_norm(bad)


@pytest.mark.parametrize("bits, what, change", [(bits, *case) for bits, test in ((32, test_step_refuses), (8, test_8_bit_step_refuses))
                                                for case in test.pytestmark[0].args[1]])
def test_a_refused_step_leaves_what_it_was_given(bits, what, change):
    """The very tensors of the call, those put in to have it refused among them: parameters, moments, scales, counts."""
    args = lists(bits=bits)
    options = dict(lr=1e-3)
    for k, f in change.items():
        x = f(args[k]) if callable(f) else f
        (args if k in args else options)[k] = args[x] if isinstance(x, str) else x
    given = [t for v in args.values() for t in (v if isinstance(v, list) else [v]) if isinstance(t, torch.Tensor) and not t.is_sparse]
    before = [t.clone() for t in given]
    with pytest.raises(ValueError):
        (optim.adamw8_step if bits == 8 else optim.adamw_step)(*[args[k] for k in (
            "params", "grads", "exp_avgs", "exp_avg_sqs", "scales", "steps") if k in args], **options)
    assert len(given) >= 8 and all(torch.equal(a, b) for a, b in zip(given, before)), what


def test_moments8_of_elements_whose_gradients_stop():
    """What rounding to the nearest code costs, as the module says it: with beta1 = 0.9 a first moment decays to the code 9
    (9 sqrt(0.9) = 8.54 rounds back to it), 0.5 % of its block's largest, and stays there; with beta2 = 0.999 no code of a
    second moment falls by its own decay (255 0.999^(1/4) = 254.94), so v stays what it was of the block's largest."""
    g = torch.full((512,), 1e-2)
    g[:8] = 1e-3                                         # these stop; the second block has none that do
    q, c, s = optim.moments8_encode(torch.zeros(512), torch.zeros(512))
    p, steps = torch.zeros(512), torch.zeros(1)
    for t in range(800):
        if t == 200:
            g[:8] = 0.0
            codes = c.clone()
        optim.adamw8_step([p], [g], [q], [c], [s], steps, lr=1e-3)
        if t >= 260:
            assert bool((q[0, :8] == 9).all()) and torch.equal(c, codes)
    before = p.clone()
    optim.adamw8_step([p], [g], [q], [c], [s], steps, lr=1e-3)
    assert 0.03 < float((before - p)[0]) / 1e-3 < 0.06   # 0.005 a over the root of 0.01 b, and a^2 = b: 5 % of lr a step
    m, v = optim.moments8_decode(q, c, s)
    assert abs(float(m[0, 0] / m[0, 8]) - (9 / 127) ** 2) < 1e-6 and float(v[0, 0] / v[0, 8]) > 0.009
    assert torch.equal(p[8:256], p[264:]) and float(p[0]) < 0          # and the others of the block are not touched by it
