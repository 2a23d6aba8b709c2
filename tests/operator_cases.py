"""What the operator tests share: tensors laid out in different ways, the operators' definitions in 64 bits, and how far a result may
be from them.

Bounds, element by element, with u the half step of a type (2^-24 fp32, 2^-11 fp16, 2^-8 bf16):
  * a sum of n products in 32 bits, in any order and with additions that may truncate, is off by at most (n + 8) 2^-23 times the
    sum of the products' sizes;
  * a result is rounded once: u times its size;
  * matmul: the activations' slopes are below 1.1; the special-function forms used for 16-bit results are off by less than 2^-20 of
    their argument, the exact ones by less than 2^-21;
  * rope: the angle is off by less than 2^-30, sincospif by two steps, and there are three roundings: 2^-21 of |x0| + |x1|;
  * attention: an error d of a score is a factor 1 + d of its probability, and so is the rounding of a probability to 16 bits
    (u of the inputs' type) and the 2^-19 that exponentials of scores up to 16 below the maximum are off (steps of 2^-24 times the
    exponent, and the exponential's own); both the weighted sum and the total are off by at most that, so the quotient by twice.
"""
import torch

from katago_b200 import capi

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
PRECISION = {"fp32": capi.PRECISION_FP32, "fp16": capi.PRECISION_FP16, "bf16": capi.PRECISION_BF16}


def half_step(dtype):
    return torch.finfo(TYPES[dtype]).eps / 2


def stream():
    return torch.cuda.current_stream().cuda_stream


def view(t):
    """kb_view of a tensor [batch][token][head][channel]."""
    assert t.shape[3] <= 1 or t.stride(3) == 1
    return capi.View(t.data_ptr(), *t.stride()[:3])


def laid_out(t, layout):
    """The same values in another memory order: dense, heads before tokens, rows in a wider buffer, from an odd element on."""
    b, n, h, d = t.shape
    if layout == "dense":
        return t.contiguous()
    if layout == "heads_first":
        return t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    if layout == "wide":
        room = torch.full((b, n, h * d + 24), float("nan"), dtype=t.dtype, device=t.device)
        y = room[..., 8:8 + h * d].unflatten(-1, (h, d))
        y.copy_(t)
        return y
    if layout == "odd":
        room = torch.full((b * n * (h * d + 3) + 5,), float("nan"), dtype=t.dtype, device=t.device)
        y = torch.as_strided(room, (b, n, h, d), (n * (h * d + 3), h * d + 3, d, 1), 1)
        y.copy_(t)
        return y
    raise ValueError(layout)


def assert_within(got, want, bound, what=""):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all(), what + ": not finite"
    over = (got - want).abs() - bound
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, f"{what}: over its bound by {worst:.3g} at {divmod(int(over.argmax()), over.shape[-1])}, {int((over > 0).sum())} of {over.numel()} elements"


# ---- matmul ----

def act64(v, act):
    if act == 1:
        return v.clamp_min(0)
    if act == 2:
        return v * torch.tanh(torch.nn.functional.softplus(v))
    if act == 3:
        return v * torch.sigmoid(v)
    if act == 12:
        return v * torch.tanh(torch.nn.functional.softplus(8 * v))
    return v


def matmul_reference(dtype, x, w, bias, act, residual):
    """The result and its bound."""
    x, w = x.double(), w.double()
    v, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        v, size = v + bias.double(), size + bias.double().abs()
    y = act64(v, act)
    bound = 1.1 * (x.shape[1] + 8) * 2.0 ** -23 * size
    if act:
        bound = bound + 2.0 ** -20 * v.abs()
    if residual is not None:
        bound = bound + 2.0 ** -24 * (y.abs() + residual.double().abs())
        y = y + residual.double()
    return y, bound + half_step(dtype) * (y.abs() + bound) + 1e-37 + (2.0 ** -25 if dtype == "fp16" else 0)


# ---- rope ----

def rope_reference(dtype, x, positions, freqs, rot, halves):
    """x [b][n][h][d], positions [b or 1][n][axes], freqs [tables][rot/2][axes]."""
    h = x.shape[2]
    angle = torch.einsum("bna,tpa->bntp", positions.double(), freqs.double()).repeat_interleave(h // freqs.shape[0], 2)
    cos, sin = angle.cos(), angle.sin()
    y = x.double().clone()
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if halves else (slice(0, rot, 2), slice(1, rot, 2))
    x0, x1 = x.double()[..., first], x.double()[..., second]
    y[..., first], y[..., second] = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    bound = torch.zeros_like(y)
    bound[..., first] = bound[..., second] = 2.0 ** -21 * (x0.abs() + x1.abs())
    turned = torch.zeros_like(y)
    turned[..., :rot] = 1
    return y, bound + turned * (half_step(dtype) * (y.abs() + bound) + (2.0 ** -25 if dtype == "fp16" else 0))


# ---- attention ----

def attention_reference(dtype, q, k, v, scale, q_lengths=None, k_lengths=None, key_mask=None, query_mask=None):
    """The result and its bound, rows from q_lengths on left out of neither."""
    b, n, h, dq = q.shape
    m, g = k.shape[1], h // k.shape[2]
    valid = torch.ones(b, m, dtype=torch.bool, device=q.device)
    if k_lengths is not None:
        valid &= torch.arange(m, device=q.device) < k_lengths[:, None]
    if key_mask is not None:
        valid &= key_mask != 0
    clean = valid[:, :, None, None]
    kd = torch.where(clean, k.double(), 0.0).repeat_interleave(g, 2)
    vd = torch.where(clean, v.double(), 0.0).repeat_interleave(g, 2)
    qd = q.double()
    s = torch.einsum("bihd,bjhd->bhij", qd, kd) * scale
    size = torch.einsum("bihd,bjhd->bhij", qd.abs(), kd.abs()) * scale
    s = s.masked_fill(~valid[:, None, None, :], float("-inf"))
    none = ~valid.any(1)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    p = torch.where(none[:, None, None, None], 0.0, p)
    y = torch.einsum("bhij,bjhd->bihd", p, vd)
    a = torch.einsum("bhij,bjhd->bihd", p, vd.abs())
    d = (dq + 8) * 2.0 ** -23 * (size * valid[:, None, None, :]).amax(-1) if m else torch.zeros(b, h, n, dtype=torch.float64, device=q.device)
    rel = 2 * (d + (half_step(dtype) if dtype != "fp32" else 0) + 2.0 ** -19 + (m + 8) * 2.0 ** -23)
    bound = a * rel.permute(0, 2, 1)[..., None]
    if query_mask is not None:
        live = (query_mask != 0)[:, :, None, None]
        y, bound = torch.where(live, y, 0.0), torch.where(live, bound, 0.0)
    return y, bound + half_step(dtype) * (y.abs() + bound) + (2.0 ** -25 if dtype == "fp16" else 0)


def attend(dtype, q, k, v, out, scale, q_lengths=None, k_lengths=None, key_mask=None, query_mask=None, workspace=None):
    """kb_cross_attention on tensors."""
    b, n, h, dq = q.shape
    sizes = (PRECISION[dtype], b, n, k.shape[1], h, k.shape[2], dq, v.shape[3])
    room = capi.cross_attention_workspace(*sizes)
    if workspace is None and room:
        workspace = torch.full((room,), 0xff, dtype=torch.uint8, device=q.device)  # NaN wherever it is read unwritten

    def at(t):
        return 0 if t is None else t.data_ptr()

    capi.cross_attention(*sizes, scale, view(q), view(k), view(v), view(out), at(q_lengths), at(k_lengths), at(key_mask), at(query_mask),
                         at(workspace), room, stream())
    return out
