"""The AdamW step, the 8-bit moments and the gradient norm in 64 bits, with bounds on how far an fp32 evaluation may be
off.  E = 2^-24 is half an fp32 ulp relative to the value, what one rounding may cost.

First moment, beta1 m + (1 - beta1) g': the two constants, the clip factor, two products and the sum round: 6 E (|b1 m| +
|c1 g'|); a decoded m adds 6 E (its q / 127, squared, times the scale).  Second moment: constant, clip factor and g' twice,
two products, sum: 8 E of a sum of positive terms; a decoded v adds 12 E.  Update: half the second moment's error in the
root (4 E, or 10 E), a root and a reciprocal good to one ulp (2 E each), the sum with eps, the bias corrections, the
products: 16 E (22 E) of its size, and the first moment's error over the denominator.  The parameter: the decay term's
three roundings, the subtraction in fp32 and one rounding to its type."""
import math

import torch

E = 2.0 ** -24
BLOCK = 256
TINY = 2.0 ** -126
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def decode64(q, c, s):
    q, c, s = q.double().cpu(), c.double().cpu(), s.double().cpu()
    return s[:, :1] * torch.sign(q) * (q / 127) ** 2, s[:, 1:] * (c / 255) ** 4


def norm64(grads):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


def step64(p, g, m, v, t, lr, betas, eps, weight_decay, factor=1.0):
    """(p, m, v) after the step that makes the count t, and the bounds of their fp32 errors; all on the CPU in 64 bits."""
    coded = isinstance(m, tuple)
    n = p.numel()
    dtype = p.dtype
    p, g = p.detach().double().cpu().reshape(-1), g.double().cpu().reshape(-1) * factor
    if coded:
        m, v = (x.reshape(-1)[:n] for x in decode64(*m))
    else:
        m, v = m.double().cpu().reshape(-1), v.double().cpu().reshape(-1)
    b1, b2 = betas
    m1 = b1 * m + (1 - b1) * g
    v1 = b2 * v + (1 - b2) * g * g
    em = (12 if coded else 6) * E * ((b1 * m).abs() + ((1 - b1) * g).abs())
    ev = (20 if coded else 8) * E * v1
    bc1 = -math.expm1(t * math.log(b1)) if b1 else 1.0
    bc2 = -math.expm1(t * math.log(b2)) if b2 else 1.0
    denom = (v1 / bc2).sqrt() + eps
    u = lr / bc1 * m1 / denom
    p1 = p - lr * weight_decay * p - u
    ep = (22 if coded else 16) * E * u.abs() + lr / bc1 * em / denom + 3 * E * (lr * weight_decay * p).abs() + E * p1.abs()
    half = torch.finfo(dtype).eps / 2
    ep = ep + (0 if dtype == torch.float32 else half * (p1.abs() + ep) + torch.finfo(dtype).smallest_normal * half)
    return (p1, m1, v1), (ep, em, ev)


def assert_near(got, want, bound, what):
    got = got.detach().double().cpu().reshape(-1)
    off = (got - want).abs()
    bad = ~(off <= bound + 1e-44)
    if bool(bad.any()):
        i = int(torch.nonzero(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {float(got[i])} for {float(want[i])}, "
                             f"bound {float(bound[i])}")


def assert_coded(q, c, s, m, v, em, ev, what):
    """Codes and scales of moments that are known to em and ev: every scale the block's largest, every code the nearest to
    some value within its error (a code is a rounding: 1e-3 of a step is left for the fp32 evaluation of 127 sqrt(x) and
    255 x^(1/4), 8 ulps of a number below 256 being 1.3e-4)."""
    nb = -(-m.numel() // BLOCK)
    pad = lambda x: torch.nn.functional.pad(x, (0, nb * BLOCK - x.numel())).view(nb, BLOCK)  # noqa: E731
    m, v, em, ev = (pad(x) for x in (m, v, em, ev))
    q, c, s = q.double().cpu(), c.double().cpu(), s.double().cpu()
    a, b = s[:, 0], s[:, 1]
    ea, eb = em.amax(1), ev.amax(1)
    assert bool(((a - m.abs().amax(1)).abs() <= ea + 1e-44).all()), what
    assert bool(((b - v.amax(1)).abs() <= eb + 1e-44).all()), what
    a, b = a[:, None], b[:, None]
    live_a, live_b = (a > 0).expand_as(m), (b > 0).expand_as(v)
    a, b = a.clamp(min=TINY), b.clamp(min=TINY)
    lo = (127 * ((m.abs() - em).clamp(min=0) / a).sqrt() - 0.5 - 1e-3).ceil().clamp(min=0)
    hi = (127 * ((m.abs() + em) / a).sqrt() + 0.5 + 1e-3).floor().clamp(max=127)
    assert bool(((q.abs() >= lo) & (q.abs() <= hi))[live_a].all()), (what, "first moment")
    assert bool((q[~live_a] == 0).all()) and bool((c[~live_b] == 0).all()), what
    assert bool((torch.sign(q) * torch.sign(m) >= 0)[m.abs() > em].all()), (what, "sign")
    lo = (255 * ((v - ev).clamp(min=0) / b) ** 0.25 - 0.5 - 1e-3).ceil().clamp(min=0)
    hi = (255 * ((v + ev) / b) ** 0.25 + 0.5 + 1e-3).floor().clamp(1, 255) * (v > 0)
    assert bool(((c >= torch.maximum(lo, (v > 1e-37).double())) & (c <= hi))[live_b].all()), (what, "second moment")


def make(numels, dtype, bits, device, seed=0, odd=False, step=3, scale=1e-3):
    """Parameters, gradients and moments of a run; odd: views that start at odd places of one buffer."""
    gen = torch.Generator().manual_seed(seed)
    total = sum(numels) + len(numels) + 1

    def views(x):
        out, at = [], 1
        for n in numels:
            out.append(x[at:at + n])
            at += n + (0 if odd else 0)
        return out

    def place(x):
        return views(x.to(device)) if odd else [t.clone() for t in views(x.to(device))]

    p = place((0.05 * torch.randn(total, generator=gen)).to(dtype))
    g0 = scale * torch.randn(total, generator=gen) * (torch.rand(total, generator=gen) > 0.1)
    g = place(g0.to(dtype))
    m0 = scale * 0.3 * torch.randn(total, generator=gen)
    v0 = scale ** 2 * (0.02 + torch.randn(total, generator=gen) ** 2)
    steps = torch.tensor([float(step + i % 3) for i in range(len(numels))], device=device)
    if bits == 32:
        return p, g, place(m0), place(v0), None, steps
    m, v, s = [], [], []
    for a, b in zip(views(m0), views(v0)):
        nb = -(-a.numel() // BLOCK)
        a, b = (torch.nn.functional.pad(x, (0, nb * BLOCK - x.numel())).view(nb, BLOCK) for x in (a, b))
        top = torch.stack([a.abs().amax(1), b.amax(1)], 1) if nb else torch.zeros(0, 2)
        m.append(((127 * (a.abs() / top[:, :1]).sqrt()).round() * a.sign()).to(torch.int8).to(device))
        v.append((255 * (b / top[:, 1:]) ** 0.25).round().to(torch.uint8).to(device))
        s.append(top.to(device))
    return p, g, m, v, s, steps


def check_step(run, numels, dtype, bits, device, odd=False, max_norm=None, seed=0, hyper=None, scale=1e-3):
    """run(params, grads, m, v, scales, steps, max_norm, **hyper) -> norm, against 64 bits for every tensor."""
    hyper = hyper or dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    p, g, m, v, s, steps = make(numels, dtype, bits, device, seed, odd, scale=scale)
    keep = [[t.clone() for t in x] for x in (p, g, m, v)] + [[t.clone() for t in s] if s is not None else None]
    counts = steps.tolist()
    norm = run(p, g, m, v, s, steps, max_norm, **hyper)
    total = norm64(keep[1])
    factor = 1.0
    if max_norm is not None:
        assert abs(float(norm) - total) <= 1.001 * E * total, (float(norm), total)
        factor = min(1.0, max_norm / (total + 1e-6))
    assert steps.tolist() == [c + 1 for c in counts]
    for i, n in enumerate(numels):
        assert torch.equal(g[i], keep[1][i]), "the gradient was written"
        m0, v0 = keep[2][i], keep[3][i]
        old = (m0, v0, keep[4][i]) if bits == 8 else m0
        (p1, m1, v1), (ep, em, ev) = step64(keep[0][i], keep[1][i], old, v0, counts[i] + 1, factor=factor, **hyper)
        if n == 0:
            continue
        assert_near(p[i], p1, ep, f"parameter {i}")
        if bits == 32:
            assert_near(m[i], m1, em, f"first moment {i}")
            assert_near(v[i], v1, ev, f"second moment {i}")
        else:
            assert_coded(m[i], v[i], s[i], m1, v1, em, ev, f"moments {i}")
