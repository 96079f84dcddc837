"""AdamW over many tensors in one call, with both moments in 32 or in 8 bits, and gradient norms (pir_adamw_step,
pir_grad_norm and pir_moments8_* in include/pir_hip.h; reference: one torch.optim.Adam per network,
render_surface.py:213-231).

  AdamW             a torch.optim.Optimizer; weight_decay=0 is torch.optim.Adam's step
  step_together     one step of several AdamW optimizers in one call, with one joint gradient norm
  adamw_step        the step itself on lists of tensors, moments in fp32
  adamw8_step       the same with the moments in 8 bits and a scale per 256 elements
  moments8_encode   fp32 / bf16 / fp16 moments -> 8-bit ones, and back: moments8_decode
  grad_norm         the 2-norm of every tensor and of all together

With t the step count of a tensor and g its gradient, times min(1, max_norm / (|g| + 1e-6)) where max_norm is given:

  m = beta1 m + (1 - beta1) g        v = beta2 v + (1 - beta2) g^2
  p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)

computed in fp32 and rounded once to p's type (fp32, bf16 or fp16; gradients have the type of their parameter).  The 8-bit
moments of 256 consecutive elements are m = a (q / 127) |q / 127| (int8 q) and v = b (c / 255)^4 (uint8 c) with a, b the
block's largest |m| and v in fp32, rounded to the nearest code, except that a v above zero keeps c >= 1.  A block whose
largest is below 2^-126 is zero (its next steps start from v = 0, up to (1 - beta2)^-1/2 times as long as in 32 bits unless
eps is 1e-15 or more, next to which such roots are nothing); one that holds an infinity or a NaN has a scale of NaN, and
a step that finds one in v sets both scales so: what a bad gradient does to its own moments in 32 bits, it does to its
block's in 8.  skip_nonfinite leaves everything as it is in a step whose joint norm is not finite in fp32.

A moment in 8 bits moves against its block's largest only once one step moves it by half a code's step.  So an element
whose gradients stop while its block goes on keeps 0.5 % of the block's largest m (code 9 with beta1 = 0.9) and its share of
the largest v (any code, with beta2 = 0.999), where in 32 bits both decay to zero: it goes on moving, a step by 5 % of lr if
its gradients were a tenth of the largest, by 40 % if a hundredth, by nearly lr if less.  Parameters whose elements get
gradients now and then (tables, rarely chosen rows) belong in 32 bits.

Step counts live on the device (fp32, one per tensor), so that a step can be captured into a HIP graph and replayed; a
learning rate that changes between replays is a one-element fp32 device tensor.  Calls enqueue work on the current stream
of the tensors' device and return without waiting.  Tensors on the CPU take the same formulas in torch operations.
"""
import ctypes
import math
from array import array

import torch

from . import _lib

BLOCK = 256                      # elements that share a scale
_TINY = 2.0 ** -126              # blocks whose largest is below this are zero
_LEAST_EPS = 1e-30               # with 8-bit moments: the step's reciprocals are the hardware's, which take what is below
                                 # 2^-126 for zero
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _hyper(lr, betas, eps, weight_decay, device):
    """Checked hyper-parameters of one group, and the address of a learning rate that stays on the device, or 0."""
    dev_lr = 0
    if isinstance(lr, torch.Tensor):
        if lr.numel() != 1:
            raise ValueError("lr: a number or a tensor of one element")
        if lr.is_cuda:
            if lr.dtype != torch.float32 or lr.device != device:
                raise ValueError("lr: a device tensor has to be float32, on the device of the parameters")
            dev_lr, lr = lr.data_ptr(), 0.0
    lr, beta1, beta2, eps, weight_decay = float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay)
    if not 0.0 <= lr < math.inf:
        raise ValueError(f"lr out of range: {lr}")
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError(f"betas out of range: {betas}")
    if not (0.0 <= eps < math.inf and 0.0 <= weight_decay < math.inf):
        raise ValueError(f"eps or weight_decay out of range: {eps}, {weight_decay}")
    return lr, beta1, beta2, eps, weight_decay, dev_lr


def _max_norm(max_norm):
    """The bound of the joint norm for the kernels: 0 = no clipping."""
    if max_norm is None:
        return 0.0
    max_norm = float(max_norm)
    if not max_norm > 0.0:
        raise ValueError(f"max_norm has to be positive: {max_norm}")
    return max_norm if max_norm < math.inf else 0.0


def _fills(shape, strides):
    """Whether elements with these strides fill one stretch of memory, each once, in some order of the dimensions."""
    want = 1
    for size, stride in sorted(((s, d) for s, d in zip(shape, strides) if s != 1), key=lambda x: x[1]):
        if stride != want:
            return False
        want *= size
    return True


def _dense(t):
    return t.is_contiguous() or _fills(t.shape, t.stride())


def _same_order(shape, a, b):
    return all(x == y for n, x, y in zip(shape, a, b) if n != 1)


def _check_orders(params, states):
    """Codes follow their parameter's order of memory as it was when they came to be ("strides", where it is recorded)."""
    for p, s in zip(params, states):
        if "scales" in s and "strides" in s and not _same_order(p.shape, p.stride(), s["strides"]):
            raise ValueError(f"the order of a parameter's memory changed: strides {p.stride()}, of its 8-bit moments {s['strides']}")


def _blocks(numel):
    return -(-numel // BLOCK)


def _check_disjoint(written, read):
    """Kernels write these tensors side by side: no byte of one may belong to another of them, or to one that is read."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), w)
                   for w, tensors in ((True, written), (False, read)) for t in tensors if t.numel())
    written_to = read_to = 0
    for start, end, w in spans:
        if start < written_to or (w and start < read_to):
            raise ValueError("tensors that the step writes: one is given twice, or overlaps another or a gradient")
        if w:
            written_to = max(written_to, end)
        else:
            read_to = max(read_to, end)


def _same_layout(p, t):
    return t.shape == p.shape and (t.stride() == p.stride() or (t.is_contiguous() and p.is_contiguous()))


def _check_eps(eps, coded):
    if coded and eps < _LEAST_EPS:
        raise ValueError(f"eps: at least {_LEAST_EPS} with 8-bit moments, not {eps}")


def _check(params, grads, exp_avgs, exp_avg_sqs, scales, steps):
    """Checks the lists of one device (steps: a tensor or a list of them); gradients that are laid out unlike their
    parameters come back as copies."""
    n = len(params)
    if not len(grads) == len(exp_avgs) == len(exp_avg_sqs) == n or (scales is not None and len(scales) != n):
        raise ValueError("params, grads and moments: lists of one length")
    dev = params[0].device
    out = []
    for i, (p, g, m, v) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs)):
        if p.dtype not in _DTYPES:
            raise ValueError(f"parameter {i}: {p.dtype} is not supported (float32, bfloat16, float16)")
        if g is None or g.layout is not torch.strided or g.dtype != p.dtype or g.shape != p.shape:
            raise ValueError(f"gradient {i}: a dense tensor of its parameter's shape and type is wanted")
        if not (p.device == dev and g.device == dev and m.device == dev and v.device == dev):
            raise ValueError(f"tensors {i}: on another device than parameter 0")
        if p.data_ptr() % p.element_size() or (g.data_ptr() % g.element_size() and _same_layout(p, g)):
            raise ValueError(f"tensors {i}: their addresses are not multiples of their type's size")
        if not p.is_contiguous() and not _dense(p):
            raise ValueError(f"parameter {i}: its elements do not fill one stretch of memory (strides {p.stride()})")
        s = scales[i] if scales is not None else None
        if s is None:
            if m.dtype != torch.float32 or v.dtype != torch.float32 or not (_same_layout(p, m) and _same_layout(p, v)):
                raise ValueError(f"moments {i}: float32 with their parameter's shape and strides are wanted")
        else:
            nb = _blocks(p.numel())
            if m.dtype != torch.int8 or v.dtype != torch.uint8 or s.dtype != torch.float32 or s.device != dev \
                    or tuple(m.shape) != (nb, BLOCK) or tuple(v.shape) != (nb, BLOCK) or tuple(s.shape) != (nb, 2) \
                    or not (m.is_contiguous() and v.is_contiguous() and s.is_contiguous()):
                raise ValueError(f"moments {i}: contiguous int8 and uint8 [{nb}, {BLOCK}] with float32 scales [{nb}, 2] are wanted")
            if (m.data_ptr() | v.data_ptr()) % 16 or s.data_ptr() % 8:
                raise ValueError(f"moments {i}: codes have to start at a multiple of 16 bytes, scales of 8")
        if g.is_neg() or not _same_layout(p, g):
            g = torch.empty_like(p, requires_grad=False).copy_(g)
        out.append(g)
    _check_disjoint([*params, *exp_avgs, *exp_avg_sqs, *(s for s in scales or () if s is not None),
                     *([steps] if isinstance(steps, torch.Tensor) else steps)], out)
    return out


_native = None


def _host():
    """(module, addresses of the library's entry points).  The extension is built with the library; nothing stands in for
    it on a GPU."""
    global _native
    if _native is None:
        L = _lib.lib()
        try:
            from . import _optim_host
        except ImportError as e:
            raise _lib.PirHipError(f"pir_amd/_optim_host.so: {e}; build it first (python -m pir_amd.build)") from e
        names = ("pir_adamw_step", "pir_adamw_workspace_bytes", "pir_grad_norm", "pir_grad_norm_workspace_bytes",
                 "pir_moments8_decode")
        _native = (_optim_host, *(ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in names))
    return _native


def _stream(dev):
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _run(params, grads, exp_avgs, exp_avg_sqs, scales, steps, groups, hypers, max_norm, skip_nonfinite, want_norm, states=None):
    """One pir_adamw_step.  steps: a tensor with one count per parameter, or a list of them; groups: index into hypers of
    each tensor, an array of int (None: all in the first); states: the optimizer's, whose codes record their order."""
    dev = params[0].device
    host, step, size, *_ = _host()
    rest = (exp_avgs, exp_avg_sqs, scales, steps, 0 if groups is None else groups.buffer_info()[0], hypers, max_norm,
            skip_nonfinite, want_norm, dev.index, _stream(dev), states)
    norm = host.adamw_step(step, size, params, grads, *rest)
    if norm is NotImplemented:
        _check_orders(params, states or ())
        grads = _check(params, grads, exp_avgs, exp_avg_sqs, scales, steps)
        norm = host.adamw_step(step, size, params, grads, *rest)
        if norm is NotImplemented:
            raise ValueError("plain tensors of one device are wanted")
    return norm


def _run_torch(params, grads, exp_avgs, exp_avg_sqs, scales, steps, groups, hypers, max_norm, skip_nonfinite, want_norm):
    """The same step in torch operations, for tensors on the CPU.  steps: the step counts, one-element tensors."""
    with torch.no_grad():
        norm, factor = None, 1.0
        if want_norm or skip_nonfinite or max_norm > 0.0:
            total = sum(g.double().square().sum() for g in grads).sqrt()
            norm = total.float()
            if max_norm > 0.0:
                factor = (max_norm / (total + 1e-6)).clamp(max=1.0).float()
            if skip_nonfinite and not torch.isfinite(norm):
                return norm
        for i, (p, g, m, v, t) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs, steps)):
            lr, beta1, beta2, eps, decay, _ = hypers[groups[i]]
            t.add_(1)
            count = float(t)
            s = scales[i] if scales is not None else None
            g = g.float() * factor
            if s is not None:
                numel = p.numel()
                codes, (m, v) = (m, v), (x.reshape(-1)[:numel] for x in _decode_torch(m, v, s))
                m, v = m.as_strided(p.shape, p.stride()), v.as_strided(p.shape, p.stride())
            m.mul_(beta1).add_(g, alpha=1.0 - beta1)
            v.mul_(beta2).add_(g * g * (1.0 - beta2))
            root = math.sqrt(-math.expm1(count * math.log(beta2))) if beta2 else 1.0
            size = lr / (-math.expm1(count * math.log(beta1)) if beta1 else 1.0)
            w = p.float()
            p.copy_(w - (lr * decay * w + size * (m / (v.sqrt() / root + eps))))
            if s is not None:
                flat = (numel,), (1,)
                new = _encode_torch(m.as_strided(*flat), v.as_strided(*flat))
                new[2][:, 0].masked_fill_(new[2][:, 1].isnan(), math.nan)
                for x, y in zip((*codes, s), new):
                    x.copy_(y)
        return norm


def _step(params, grads, exp_avgs, exp_avg_sqs, scales, steps, lr, betas, eps, weight_decay, max_norm, skip_nonfinite):
    params, grads = list(params), list(grads)
    bound = _max_norm(max_norm)
    want = max_norm is not None
    dev = steps.device
    hyper = _hyper(lr, betas, eps, weight_decay, dev)
    _check_eps(hyper[3], scales is not None)
    if steps.dtype != torch.float32 or not steps.is_contiguous() or steps.numel() != len(params):
        raise ValueError("steps: a contiguous float32 tensor with one count per parameter")
    if not params:
        return torch.zeros((), device=dev) if want or skip_nonfinite else None
    if params[0].device != dev:
        raise ValueError("steps: on another device than the parameters")
    if hyper[5] and dev.type != "cuda":
        raise ValueError("lr: on another device than the parameters")
    if dev.type != "cuda":
        grads = _check(params, grads, exp_avgs, exp_avg_sqs, scales, steps)
        return _run_torch(params, grads, exp_avgs, exp_avg_sqs, scales, list(steps.view(-1)), [0] * len(params), [hyper],
                          bound, skip_nonfinite, want)
    return _run(params, grads, list(exp_avgs), list(exp_avg_sqs), scales, steps, None, [hyper], bound, skip_nonfinite, want)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0,
               max_norm=None, skip_nonfinite=False):
    """One AdamW step, in place, of lists of tensors on one device; moments are fp32 with their parameter's shape and
    strides, steps is fp32 [len(params)], all of it zero before the first step.  None of what the step writes may share
    memory with another tensor of the call.  Returns the joint gradient norm (before clipping; a 0-dim device tensor) with
    max_norm (inf: not clipped) or skip_nonfinite, else None."""
    return _step(params, grads, exp_avgs, exp_avg_sqs, None, steps, lr, betas, eps, weight_decay, max_norm, skip_nonfinite)


def adamw8_step(params, grads, exp_avgs, exp_avg_sqs, scales, steps, *, lr, betas=(0.9, 0.999), eps=1e-8,
                weight_decay=0.0, max_norm=None, skip_nonfinite=False):
    """adamw_step with 8-bit moments: of a parameter of n elements, exp_avg is int8 [ceil(n / 256), 256], exp_avg_sq uint8
    of that shape and scales fp32 [ceil(n / 256), 2]; elements count in the order of memory."""
    return _step(params, grads, exp_avgs, exp_avg_sqs, list(scales), steps, lr, betas, eps, weight_decay, max_norm,
                 skip_nonfinite)


def _check_norm(tensors, dev):
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPES or t.layout is not torch.strided or t.device != dev:
            raise ValueError(f"tensor {i}: dense float32, bfloat16 or float16 on the device of tensor 0 is wanted")


def grad_norm(tensors):
    """(total, each): the 2-norm of all tensors together (0-dim) and of every one ([len(tensors)]), fp32 tensors on their
    device.  Squares and sums in 64 bits; the same bits on every run."""
    tensors = list(tensors)
    if not tensors:
        raise ValueError("grad_norm: no tensors")
    dev = getattr(tensors[0], "device", None)
    with torch.no_grad():
        if dev is None or dev.type != "cuda":
            _check_norm(tensors, dev)
            each = torch.stack([t.double().square().sum() for t in tensors])
            return each.sum().sqrt().float(), each.sqrt().float()
        host, _, _, norm, size, _ = _host()
        out = host.grad_norm(norm, size, tensors, dev.index, _stream(dev))
        if out is NotImplemented:
            _check_norm(tensors, dev)
            tensors = [t.resolve_neg() if _dense(t) else t.contiguous() for t in tensors]
            out = host.grad_norm(norm, size, tensors, dev.index, _stream(dev))
            if out is NotImplemented:
                raise ValueError("plain tensors of one device are wanted")
    return out[0], out[1:]


# ------------------------------------------------------------------------------------------------ 8-bit moments
def _decode_torch(exp_avg, exp_avg_sq, scales):
    q, c = exp_avg.float() / 127, exp_avg_sq.float() / 255
    c = c * c
    return scales[:, :1] * (q * q.abs()), scales[:, 1:] * (c * c)


def _encode_torch(m, v):
    numel = m.numel()
    nb = _blocks(numel)
    m, v = (torch.nn.functional.pad(x.reshape(-1).float(), (0, nb * BLOCK - numel)).view(nb, BLOCK) for x in (m, v))
    scales = torch.stack([m.abs().amax(1), v.abs().amax(1)], 1)
    scales = torch.where(torch.isfinite(scales), torch.where(scales < _TINY, 0.0, scales), math.nan)
    a, b = scales[:, :1], scales[:, 1:]
    q = torch.where(a > 0, (127 * (m.abs() / a).sqrt()).round() * m.sign(), 0.0)
    c = torch.where((b > 0) & (v > 0), (255 * (v / b).sqrt().sqrt()).round().clamp(min=1), 0.0)
    return q.to(torch.int8), c.to(torch.uint8), scales


def moments8_encode(exp_avg, exp_avg_sq):
    """Moments of one tensor (float32, bfloat16 or float16, both of one shape, strides and type) -> (int8 codes, uint8
    codes, scales) as adamw8_step takes them."""
    m, v = exp_avg, exp_avg_sq
    if m.dtype not in _DTYPES or v.dtype != m.dtype or m.device != v.device or not _same_layout(m, v):
        raise ValueError("moments: float32, bfloat16 or float16, both of one type, shape, strides and device")
    if not _dense(m):
        raise ValueError("moments: their elements do not fill one stretch of memory")
    with torch.no_grad():
        numel, nb, dev = m.numel(), _blocks(m.numel()), m.device
        if dev.type != "cuda":
            return _encode_torch(m.as_strided((numel,), (1,)), v.as_strided((numel,), (1,)))
        m, v = m.resolve_neg(), v.resolve_neg()
        out = (torch.empty(nb, BLOCK, dtype=torch.int8, device=dev), torch.empty(nb, BLOCK, dtype=torch.uint8, device=dev),
               torch.empty(nb, 2, dtype=torch.float32, device=dev))
        with torch.cuda.device(dev):
            _lib.check(_lib.lib().pir_moments8_encode(numel, _DTYPES[m.dtype], m.data_ptr(), v.data_ptr(),
                                                      *[t.data_ptr() for t in out], _stream(dev)), "pir_moments8_encode")
        return out


def moments8_decode(exp_avg, exp_avg_sq, scales, dtype=torch.float32):
    """8-bit moments of any number of blocks -> (exp_avg, exp_avg_sq) as values of dtype, [blocks, 256] each."""
    q, c, s = exp_avg, exp_avg_sq, scales
    if dtype not in _DTYPES:
        raise ValueError(f"dtype: {dtype} is not supported (float32, bfloat16, float16)")
    if q.is_cuda:
        host, *_, decode = _host()
        out = host.moments8_decode(decode, q, c, s, _DTYPES[dtype], q.device.index, _stream(q.device))
        if out is not NotImplemented:
            return out
    if q.dtype != torch.int8 or c.dtype != torch.uint8 or s.dtype != torch.float32 or q.dim() != 2 or q.shape[1] != BLOCK \
            or c.shape != q.shape or tuple(s.shape) != (q.shape[0], 2) or not (q.device == c.device == s.device) \
            or not (q.is_contiguous() and c.is_contiguous() and s.is_contiguous()):
        raise ValueError("moments: contiguous int8 and uint8 [blocks, 256] with float32 scales [blocks, 2] are wanted")
    if q.is_cuda:
        raise ValueError("moments: codes have to start at a multiple of 16 bytes, scales of 8")
    return tuple(x.to(dtype) for x in _decode_torch(q, c, s))


# ------------------------------------------------------------------------------------------------- the optimizer
class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's step (weight_decay=0: torch.optim.Adam's) in one call for all parameters of a device.

    state_bits=8 keeps the moments of parameters of at least min_8bit_numel elements in 8 bits (2.03 bytes a parameter in
    place of 8); smaller ones, biases above all, stay in 32.  max_norm clips the joint gradient norm of the optimizer's
    parameters inside the step, without a pass of its own; skip_nonfinite leaves parameters, moments and step counts as
    they are in a step whose joint norm is not finite.  Either leaves the norm before clipping in total_norm, a
    device tensor.  A parameter without a gradient is skipped: no state, no step counted.

    state[p]: "step" (fp32, on p's device), "exp_avg", "exp_avg_sq" and, in 8 bits, "scales" and the "strides" of p, whose
    order of memory the codes follow.  load_state_dict takes the states of torch.optim.Adam and AdamW too, and converts
    between 32 and 8 bits as this optimizer's groups ask for, and between orders of memory."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, min_8bit_numel=4096,
                 max_norm=None, skip_nonfinite=False):
        _max_norm(max_norm)
        self.max_norm, self.skip_nonfinite, self.total_norm = max_norm, skip_nonfinite, None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_numel=min_8bit_numel))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        g = self.param_groups[-1]
        try:
            _hyper(g["lr"], g["betas"], g["eps"], g["weight_decay"], g["params"][0].device if g["params"] else None)
            if g["state_bits"] not in (32, 8):
                raise ValueError(f"state_bits has to be 32 or 8: {g['state_bits']}")
        except ValueError:
            self.param_groups.pop()
            raise

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm, "skip_nonfinite": self.skip_nonfinite, "total_norm": None}

    def __setstate__(self, state):
        super().__setstate__(state)
        for g in self.param_groups:
            for k, v in self.defaults.items():
                g.setdefault(k, v)

    @staticmethod
    def _in_8_bits(p, group):
        return group["state_bits"] == 8 and p.numel() >= group["min_8bit_numel"]

    def _new_state(self, p, group):
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a parameter's first step cannot be captured: every replay would clear its moments; take "
                               "one step before the capture")
        s = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
        if self._in_8_bits(p, group):
            nb = _blocks(p.numel())
            s["exp_avg"] = torch.zeros(nb, BLOCK, dtype=torch.int8, device=p.device)
            s["exp_avg_sq"] = torch.zeros(nb, BLOCK, dtype=torch.uint8, device=p.device)
            s["scales"] = torch.zeros(nb, 2, dtype=torch.float32, device=p.device)
            s["strides"] = p.stride()
        else:
            for k in ("exp_avg", "exp_avg_sq"):
                s[k] = torch.zeros_like(p, dtype=torch.float32, requires_grad=False, memory_format=torch.preserve_format)
        return s

    def _state_of(self, p, group):
        s = self.state[p]
        if not s:
            s.update(self._new_state(p, group))
        return s

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self.total_norm = step_together([self], self.max_norm, self.skip_nonfinite)
        return loss

    def load_state_dict(self, state_dict):
        """Takes what state_dict() of this class, torch.optim.Adam or torch.optim.AdamW returns; state_bits and min_8bit_numel
        of the groups stay this optimizer's, and the moments are converted to them.  What cannot be taken is refused before
        anything changes."""
        own = [{k: g[k] for k in ("state_bits", "min_8bit_numel")} for g in self.param_groups]
        states = {}

        def convert(_, d):       # the last before the load: sees what other hooks put in place
            for g in d["param_groups"]:
                if g.get("amsgrad") or g.get("maximize"):
                    raise ValueError("amsgrad and maximize are not supported")
                if g.get("weight_decay") and not g.get("decoupled_weight_decay", True):
                    raise ValueError("the weight decay of torch.optim.Adam (added to the gradient) is not supported")
            if [len(g["params"]) for g in d["param_groups"]] == [len(g["params"]) for g in self.param_groups]:
                ids = (i for g in d["param_groups"] for i in g["params"])
                for i, (p, g) in zip(ids, [(p, g) for g in self.param_groups for p in g["params"]]):
                    if d["state"].get(i):
                        states[p] = self._converted(i, p, g, d["state"][i])
            return {**d, "state": {}}            # the load itself would cast codes to the parameters' type

        def put(_):              # the first after it
            for g, bits in zip(self.param_groups, own):
                g.update(bits)
            self.state.update(states)
        hooks = (self.register_load_state_dict_pre_hook(convert), self.register_load_state_dict_post_hook(put, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @torch.no_grad()
    def _converted(self, i, p, group, saved):
        """A state of p, in its group's number of bits, of the saved one."""
        for k in ("step", "exp_avg", "exp_avg_sq"):
            if k not in saved:
                raise ValueError(f"state of parameter {i}: {k} is missing")
        put = {k: saved[k].detach().to(p.device) for k in ("exp_avg", "exp_avg_sq", "scales") if k in saved}
        nb = _blocks(p.numel())
        coded = {"exp_avg": (nb, BLOCK), "exp_avg_sq": (nb, BLOCK), "scales": (nb, 2)}
        types = {"exp_avg": torch.int8, "exp_avg_sq": torch.uint8, "scales": torch.float32}
        for k, x in put.items():
            want = coded[k] if "scales" in put else tuple(p.shape)
            if tuple(x.shape) != want:
                raise ValueError(f"state of parameter {i}: {k} of shape {tuple(x.shape)} for a parameter of {tuple(p.shape)}")
            if x.dtype != types[k] if "scales" in put else not x.is_floating_point():
                raise ValueError(f"state of parameter {i}: {k} of type {x.dtype}")
        order = saved.get("strides", p.stride())
        if "scales" in put:
            if "strides" not in saved and not p.is_contiguous():
                raise ValueError(f"state of parameter {i}: the order of its codes is not recorded, and the parameter not contiguous")
            if not isinstance(order, (tuple, list)) or len(order) != p.dim() or not all(isinstance(x, int) for x in order) \
                    or (p.numel() and not _fills(p.shape, order)):
                raise ValueError(f"state of parameter {i}: strides {order} are no order of a parameter of {tuple(p.shape)}")
        s = self._new_state(p, group)
        s["step"].fill_(float(saved["step"]))
        if "scales" in put and not ("scales" in s and _same_order(p.shape, order, p.stride())):
            m, v = moments8_decode(*(put[k].contiguous() for k in ("exp_avg", "exp_avg_sq", "scales")))
            put = {k: x.reshape(-1)[:p.numel()].as_strided(p.shape, order) for k, x in (("exp_avg", m), ("exp_avg_sq", v))}
        if "scales" in s and "scales" not in put:
            like = torch.empty_like(p, dtype=torch.float32, requires_grad=False)
            m, v = (like.clone().copy_(put[k]) for k in ("exp_avg", "exp_avg_sq"))
            put = dict(zip(("exp_avg", "exp_avg_sq", "scales"), moments8_encode(m, v)))
        for k, x in put.items():
            s[k].copy_(x)
        return s


@torch.no_grad()
def step_together(optimizers, max_norm=None, skip_nonfinite=False):
    """One step of several AdamW optimizers in one call, their gradients clipped to one joint norm.  (The optimizers' own
    max_norm and skip_nonfinite are for their own step().)  Returns the joint norm with max_norm or skip_nonfinite."""
    bound = _max_norm(max_norm)
    parts = []                   # the tensors of one group on one device
    for opt in optimizers:
        if not isinstance(opt, AdamW):
            raise TypeError(f"step_together takes pir_amd.optim.AdamW optimizers, not {type(opt).__name__}")
        for group in opt.param_groups:
            live = [p for p in group["params"] if p.grad is not None]
            places = {p.get_device() for p in live}
            for place in places:
                parts.append((place, opt, group, live if len(places) == 1 else [p for p in live if p.get_device() == place]))
    if (max_norm is not None or skip_nonfinite) and len({place for place, *_ in parts}) > 1:
        raise ValueError("a joint norm of parameters on several devices is not supported")
    jobs = {}                    # device -> its tensors, of all optimizers
    for place, opt, group, mine in parts:
        states = [opt.state[p] for p in mine]
        if not all(states):
            states = [opt._state_of(p, group) for p in mine]
        job = jobs.setdefault(place, _Job(mine[0].device))
        job.add(mine, states, _hyper(group["lr"], group["betas"], group["eps"], group["weight_decay"], job.device))
    norm = torch.zeros(()) if max_norm is not None or skip_nonfinite else None      # what no gradients have
    for job in jobs.values():
        norm = job.run(bound, skip_nonfinite, max_norm is not None)
    return norm


class _Job:
    """The tensors of one device in a step of one or more optimizers."""

    def __init__(self, device):
        self.device, self.params, self.states, self.groups, self.hypers = device, [], [], array("i"), []

    def add(self, params, states, hyper):
        if hyper[5] and self.device.type != "cuda":
            raise ValueError("lr: on another device than the parameters")
        if hyper[3] < _LEAST_EPS:
            _check_eps(hyper[3], any("scales" in s for s in states))
        self.params += params
        self.states += states
        self.groups.extend([len(self.hypers)] * len(params))
        self.hypers.append(hyper)

    def run(self, bound, skip_nonfinite, want_norm):
        grads = [p.grad for p in self.params]
        m, v, t = ([s[k] for s in self.states] for k in ("exp_avg", "exp_avg_sq", "step"))
        scales = [s.get("scales") for s in self.states]
        rest = (t, self.groups, self.hypers, bound, skip_nonfinite, want_norm)
        if self.device.type == "cuda":
            return _run(self.params, grads, m, v, scales, *rest, self.states)
        _check_orders(self.params, self.states)
        return _run_torch(self.params, _check(self.params, grads, m, v, scales, t), m, v, scales, *rest)
