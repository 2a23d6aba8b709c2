"""The transformer operators on a caller's own device buffers, as cases for timing and comparison.

kb_matmul (product with bias, activation and residual), kb_rope (rotary positions with several axes) and
kb_cross_attention (attention to states of another length) are the parts of one block that lets a net's tokens look at
an encoder's states: earlier positions of a game, a text, a video.  `listed` names ordinary calls, `draw` gives others of
the same ranges, `prepare` makes what a program holds before the call, `run` is the call, `exact` the operator's
definition in 64 bits.  With `own` false `run` computes the operators in elementary torch operations.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_PRECISIONS = {"fp32": 0, "fp16": 1, "bf16": 2}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
_ACTS = {"identity": 0, "relu": 1, "mish": 2, "silu": 3}


# ---- cases ----

def _matmul(dtype, m, n, k, act="identity", bias=False, residual=False, **more):
    return dict(more, op="matmul", dtype=dtype, m=m, n=n, k=k, act=act, bias=bias, residual=residual)


def _rope(dtype, batch, tokens, q_heads, k_heads, dim, rot, axes, halves, places, **more):
    return dict(more, op="rope", dtype=dtype, batch=batch, tokens=tokens, q_heads=q_heads, k_heads=k_heads, dim=dim, rot=rot, axes=axes,
                halves=halves, places=places)


def _attention(dtype, batch, q_len, k_len, heads, kv_heads, qk_dim, v_dim, ragged=False, mask=False, **more):
    return dict(more, op="attention", dtype=dtype, batch=batch, q_len=q_len, k_len=k_len, heads=heads, kv_heads=kv_heads, qk_dim=qk_dim,
                v_dim=v_dim, ragged=ragged, mask=mask)


def listed():
    return [
        # the projection of a few sequences' newest tokens: the weights are what is read
        _matmul("bf16", 4, 4096, 4096, bias=True, residual=True, name="matmul_few_tokens"),
        # the first half of a feed-forward layer over a full batch of 19x19 boards
        _matmul("fp16", 46208, 1024, 384, act="silu", bias=True, name="matmul_board_batch"),
        # three boards in the exact type, from one point per column to the 362 logits of a policy
        _matmul("fp32", 1083, 362, 361, act="mish", bias=True, residual=True, name="matmul_fp32_odd"),
        # an output projection with its residual over many tokens
        _matmul("bf16", 8192, 4096, 4096, residual=True, name="matmul_large"),
        # the newest token of one game record
        _rope("fp16", 1, 1, 6, 6, 64, 64, 2, False, "far", name="rope_one_token"),
        # the points of a full batch of 19x19 boards by row and column, which all boards share
        _rope("fp16", 128, 361, 6, 6, 64, 64, 2, False, "shared", name="rope_board_batch"),
        # two clips: time, height, width; grouped keys
        _rope("bf16", 2, 13 * 30 * 52, 24, 8, 128, 128, 3, True, "grid", name="rope_video"),
        # boards of several past turns in the exact type; a part of each head has no position
        _rope("fp32", 7, 1083, 5, 5, 80, 48, 3, False, "grid", name="rope_fp32_partial"),
        # the points of a board look at the points of up to eight earlier positions of their game (a first position has none)
        _attention("fp16", 64, 361, 2888, 6, 6, 64, 64, ragged=True, mask=True, name="attention_history"),
        # one new token of each of eight sequences over the kept keys and values of a long input
        _attention("bf16", 8, 1, 32768, 32, 8, 128, 128, ragged=True, name="attention_one_token"),
        # many tokens over a longer input, every key valid
        _attention("bf16", 2, 4096, 8192, 16, 16, 128, 128, name="attention_large"),
        # grouped heads of 32 and 16 channels in the exact type over a short text
        _attention("fp32", 8, 1521, 77, 8, 4, 32, 16, ragged=True, name="attention_fp32_text"),
    ]


def _between(rng, least, most):
    """Whole numbers spread over the logarithm of a range, odd ones as often as even ones."""
    return min(most, max(least, round(least * (most / least) ** rng.random())))


def draw(rng):
    op = rng.choice(("matmul", "rope", "attention"))
    dtype = rng.choice(("fp16", "fp16", "bf16", "bf16", "fp32"))
    if op == "matmul":
        while True:
            m, n, k = _between(rng, 1, 50000), _between(rng, 16, 8192), _between(rng, 16, 8192)
            if rng.random() < 0.7:  # most widths are whole vectors
                n, k = (n + 7) // 8 * 8, (k + 7) // 8 * 8
            if m * n * k <= (1 << 35 if dtype == "fp32" else 1 << 37) and m * (n + k) <= 1 << 27:
                return _matmul(dtype, m, n, k, act=rng.choice(sorted(_ACTS)), bias=rng.random() < 0.6, residual=rng.random() < 0.5)
    if op == "rope":
        dim = rng.choice((32, 48, 64, 80, 96, 128))
        rot = rng.choice((dim, dim, dim // 2))
        k_heads = rng.choice((1, 2, 4, 6, 8))
        q_heads = k_heads * rng.choice((1, 1, 2, 4))
        while True:
            batch, tokens = _between(rng, 1, 256), _between(rng, 1, 20000)
            if batch * tokens * (q_heads + k_heads) * dim <= 1 << 27:
                return _rope(dtype, batch, tokens, q_heads, k_heads, dim, rot, rng.choice((1, 2, 3)), rng.random() < 0.5,
                             rng.choice(("shared", "grid", "far")))
    qk_dim = rng.choice((16, 32, 48, 64, 64, 80, 96, 128, 128))
    v_dim = rng.choice((qk_dim, qk_dim, qk_dim, 64))
    kv_heads = rng.choice((1, 2, 4, 6, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 8))
    while True:
        batch, q_len, k_len = _between(rng, 1, 64), rng.choice((1, _between(rng, 1, 4096), _between(rng, 1, 4096))), _between(rng, 1, 32768)
        pairs = batch * heads * q_len * k_len
        if pairs <= (1 << 28 if dtype == "fp32" else 1 << 30) and batch * k_len * kv_heads * (qk_dim + v_dim) <= 1 << 29:
            return _attention(dtype, batch, q_len, k_len, heads, kv_heads, qk_dim, v_dim, ragged=rng.random() < 0.5, mask=rng.random() < 0.3)


def _lengths(case):
    """Valid keys of each sequence: spread from none to all where the batch is ragged."""
    batch, most = case["batch"], case["k_len"]
    if not case["ragged"]:
        return [most] * batch
    return [(most * i + batch - 2) // (batch - 1) for i in range(batch)] if batch > 1 else [(most + 1) // 2]


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": e * (m * k + n * k + m * n * (2 if case["residual"] else 1)) + (4 * n if case["bias"] else 0), "flops": 2.0 * m * n * k}
    if case["op"] == "rope":
        rows = case["batch"] * case["tokens"] * (case["q_heads"] + case["k_heads"])
        places = case["tokens"] * (1 if case["places"] == "shared" else case["batch"]) * case["axes"]
        return {"bytes": 2 * e * rows * case["dim"] + 4 * places, "flops": 3.0 * rows * case["rot"]}
    keys = sum(_lengths(case))
    width = case["qk_dim"] + case["v_dim"]
    return {"bytes": e * width * (case["batch"] * case["q_len"] * case["heads"] + keys * case["kv_heads"]) + (4 * keys if case["mask"] else 0),
            "flops": 2.0 * case["q_len"] * keys * case["heads"] * width}


# ---- inputs ----

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=t):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(scale)

    s = dict(case=case)
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"], s["w"] = normal(m, k), normal(n, k, scale=k ** -0.5)
        s["bias"] = normal(n, scale=0.5, dtype=torch.float32) if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
        s["y"] = torch.empty(m, n, device="cuda", dtype=t)
        return s
    if case["op"] == "rope":
        b, n, d, a, pairs = case["batch"], case["tokens"], case["dim"], case["axes"], case["rot"] // 2
        s["q"], s["k"] = normal(b, n, case["q_heads"], d), normal(b, n, case["k_heads"], d)
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        # each pair turns with one axis, every axis has its own geometric series; a third of the tables is learned and mixes them
        freqs = torch.zeros(pairs, a, device="cuda", dtype=torch.float64)
        for axis in range(a):
            mine = torch.arange(axis, pairs, a, device="cuda")
            freqs[mine, axis] = 10000.0 ** (-torch.arange(len(mine), device="cuda", dtype=torch.float64) / max(1, len(mine)))
        s["freqs"] = (freqs.float() * (1 + 0.05 * normal(pairs, a, dtype=torch.float32))).contiguous()
        rows = 1 if case["places"] == "shared" else b
        i = torch.arange(n, device="cuda")
        width = max(1, math.isqrt(n))
        place = torch.stack([i // (width * 8), i // width, i % width][-a:] if a > 1 else [i], -1).expand(rows, n, a)
        if case["places"] != "shared":  # sequences begin anywhere: near zero, or deep in a long input
            first = torch.randint(0, 1 << 20 if case["places"] == "far" else 64, (rows, 1, a), generator=g, device="cuda")
            place = place + first
        s["places"] = place.to(torch.int32).contiguous()
        return s
    b, h, hk, dq, dv = case["batch"], case["heads"], case["kv_heads"], case["qk_dim"], case["v_dim"]
    s["q"] = normal(b, case["q_len"], h, dq)
    # one projection writes keys and values side by side
    kv = normal(b, case["k_len"], hk * (dq + dv))
    s["k"] = kv[..., :hk * dq].view(b, case["k_len"], hk, dq)
    s["v"] = kv[..., hk * dq:].view(b, case["k_len"], hk, dv)
    s["out"] = torch.empty(b, case["q_len"], h, dv, device="cuda", dtype=t)
    s["lengths"] = None
    if case["ragged"]:
        order = torch.randperm(b, generator=g, device="cuda")
        s["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[order].contiguous()
    s["mask"] = None
    if case["mask"]:  # points off a smaller board, padding between parts
        s["mask"] = (torch.rand(b, case["k_len"], generator=g, device="cuda") < 0.8).float()
    return s


# ---- one pass ----

def run(state):
    return _RUN[state["case"]["op"]](state, state["case"])


def _act(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "mish":
        return v * torch.tanh(v.clamp_min(0) + torch.log1p(torch.exp(-v.abs())))
    return v


def _run_matmul(s, c):
    x, w, y, bias, residual = s["x"], s["w"], s["y"], s["bias"], s["residual"]
    if own:
        from katago_b200 import capi
        capi.matmul(_PRECISIONS[c["dtype"]], c["m"], c["n"], c["k"], x.data_ptr(), c["k"], w.data_ptr(), c["k"], y.data_ptr(), c["n"],
                    bias=bias.data_ptr() if bias is not None else 0, act=_ACTS[c["act"]],
                    residual=residual.data_ptr() if residual is not None else 0, ldr=c["n"], stream=torch.cuda.current_stream().cuda_stream)
        return y
    v = x.float() @ w.float().t()
    if bias is not None:
        v = v + bias
    v = _act(v, c["act"])
    if residual is not None:
        v = v + residual.float()
    return v.to(x.dtype)


def _run_rope(s, c):
    q, k, places, freqs = s["q"], s["k"], s["places"], s["freqs"]
    if own:
        from katago_b200 import capi
        view = capi.View
        capi.rope(_PRECISIONS[c["dtype"]], c["batch"], c["tokens"], c["dim"], c["rot"], places.data_ptr(),
                  0 if c["places"] == "shared" else c["tokens"] * c["axes"], c["axes"], freqs.data_ptr(), 1, int(c["halves"]),
                  view(q.data_ptr(), *q.stride()[:3]), view(s["q_out"].data_ptr(), *q.stride()[:3]), c["q_heads"],
                  view(k.data_ptr(), *k.stride()[:3]), view(s["k_out"].data_ptr(), *k.stride()[:3]), c["k_heads"],
                  stream=torch.cuda.current_stream().cuda_stream)
        return s["q_out"], s["k_out"]
    angle = (places.double()[:, :, None, :] * freqs.double()).sum(-1)  # [rows][tokens][pairs]
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    return tuple(_turned(x, cos, sin, c["rot"], c["halves"]) for x in (q, k))


def _turned(x, cos, sin, rot, halves):
    v = x[..., :rot].float()
    a, b = (v[..., :rot // 2], v[..., rot // 2:]) if halves else (v[..., 0::2], v[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    v = torch.cat((a, b), -1) if halves else torch.stack((a, b), -1).flatten(-2)
    return torch.cat((v.to(x.dtype), x[..., rot:]), -1)


def _run_attention(s, c):
    q, k, v, lengths, mask = s["q"], s["k"], s["v"], s["lengths"], s["mask"]
    if own:
        from katago_b200 import capi
        view, out, precision = capi.View, s["out"], _PRECISIONS[c["dtype"]]
        room = capi.cross_attention_workspace(precision, c["batch"], c["q_len"], c["k_len"], c["heads"], c["kv_heads"], c["qk_dim"], c["v_dim"])
        space = torch.empty(room, dtype=torch.uint8, device="cuda") if room else None
        capi.cross_attention(precision, c["batch"], c["q_len"], c["k_len"], c["heads"], c["kv_heads"], c["qk_dim"], c["v_dim"], c["qk_dim"] ** -0.5,
                             view(q.data_ptr(), *q.stride()[:3]), view(k.data_ptr(), *k.stride()[:3]), view(v.data_ptr(), *v.stride()[:3]),
                             view(out.data_ptr(), *out.stride()[:3]), k_lengths=lengths.data_ptr() if lengths is not None else 0,
                             key_mask=mask.data_ptr() if mask is not None else 0, workspace=space.data_ptr() if room else 0, workspace_bytes=room,
                             stream=torch.cuda.current_stream().cuda_stream)
        return out
    b, n, h, dq = q.shape
    hk, m, dv = k.shape[2], k.shape[1], v.shape[3]
    rows = q.float().view(b, n, hk, h // hk, dq).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, dq)  # a key head's rows together
    score = (rows @ k.float().permute(0, 2, 3, 1)) * dq ** -0.5
    if lengths is not None or mask is not None:
        valid = torch.ones(b, m, dtype=torch.bool, device=q.device)
        if lengths is not None:
            valid &= torch.arange(m, device=q.device) < lengths[:, None]
        if mask is not None:
            valid &= mask != 0
        score = torch.where(valid[:, None, None, :], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    out = (p @ v.float().permute(0, 2, 1, 3)) / torch.where(total > 0, total, 1.0)
    return out.view(b, hk, h // hk, n, dv).permute(0, 3, 1, 2, 4).reshape(b, n, h, dv).to(q.dtype)


_RUN = {"matmul": _run_matmul, "rope": _run_rope, "attention": _run_attention}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "matmul":
        y = torch.einsum("mk,nk->mn", s["x"].double(), s["w"].double())
        if case["bias"]:
            y += s["bias"].double()[None]
        if case["act"] == "relu":
            y = torch.maximum(y, torch.zeros_like(y))
        elif case["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["act"] == "mish":
            y = y * torch.tanh(torch.logaddexp(y, torch.zeros_like(y)))
        return y + s["residual"].double() if case["residual"] else y
    if case["op"] == "rope":
        turn = torch.zeros(*s["places"].shape[:2], case["rot"] // 2, dtype=torch.float64, device="cuda")
        for axis in range(case["axes"]):
            turn += torch.outer(s["places"][..., axis].double().flatten(), s["freqs"][:, axis].double()).view_as(turn)
        unit = torch.polar(torch.ones_like(turn), turn)[:, :, None]
        found = []
        for x in (s["q"], s["k"]):
            y = x.double()
            if case["halves"]:
                z = torch.complex(y[..., :case["rot"] // 2], y[..., case["rot"] // 2:case["rot"]]) * unit
                y[..., :case["rot"] // 2], y[..., case["rot"] // 2:case["rot"]] = z.real, z.imag
            else:
                z = torch.complex(y[..., 0:case["rot"]:2], y[..., 1:case["rot"]:2]) * unit
                y[..., 0:case["rot"]:2], y[..., 1:case["rot"]:2] = z.real, z.imag
            found.append(y)
        return tuple(found)
    b, n, h, group = case["batch"], case["q_len"], case["heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(b, n, h, case["v_dim"], dtype=torch.float64, device="cuda")
    for i in range(b):
        keys = torch.arange(case["k_len"], device="cuda")
        if case["ragged"]:
            keys = keys[:int(s["lengths"][i])]
        if case["mask"]:
            keys = keys[s["mask"][i, keys] != 0]
        if not len(keys):
            continue
        for kv in range(case["kv_heads"]):
            k, v = s["k"][i, keys, kv].double(), s["v"][i, keys, kv].double()
            q = s["q"][i, :, kv * group:(kv + 1) * group].double() / math.sqrt(case["qk_dim"])
            for j in range(0, n, 1024):
                p = torch.softmax(torch.einsum("ngd,kd->ngk", q[j:j + 1024], k), -1)
                out[i, j:j + 1024, kv * group:(kv + 1) * group] = torch.einsum("ngk,kd->ngd", p, v)
    return out
