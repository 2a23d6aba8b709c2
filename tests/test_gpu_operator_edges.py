"""kb_matmul, kb_rope and kb_cross_attention where their arithmetic ends: infinities, NaN, weights and angles at the edge of a type; and
calls that share memory or a graph in unusual ways.  (Bounds: operator_cases.py.)"""
import ctypes
import math
import threading
from fractions import Fraction

import pytest

torch = pytest.importorskip("torch")

from katago_b200 import capi  # noqa: E402
from tests.operator_cases import PRECISION, TYPES, assert_within, attend, attention_reference, matmul_reference, stream, view  # noqa: E402
from tests.test_gpu_operators import ALL, NAN, attention_inputs, empty_out, multiply, normal, seeded, turn  # noqa: E402

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

INF = float("inf")


# ---- memory that a call's tensors share ----

def test_inputs_that_repeat_beside_the_output_in_one_buffer():
    """A query that all tokens of a sequence share, interleaved with the output: refused, since its rows are further apart than the
    output's.  In a buffer of its own it is taken."""
    fp32 = PRECISION["fp32"]
    whole = torch.zeros(2, 1 + 8, 64, device="cuda")
    at, step = whole.data_ptr(), 9 * 64
    repeated, out = capi.View(at, step, 0, 64), capi.View(at + 4 * 64, step, 64, 64)
    pos, freqs = torch.zeros(8, 1, dtype=torch.int32, device="cuda"), torch.zeros(32, 1, device="cuda")
    with pytest.raises(capi.KBError, match="q out overlaps q in"):
        capi.rope(fp32, 2, 8, 64, 64, pos.data_ptr(), 0, 1, freqs.data_ptr(), 1, 0, repeated, out, 1, stream=stream())
    kv = torch.ones(2, 5, 1, 64, device="cuda")
    with pytest.raises(capi.KBError, match="out overlaps q"):
        capi.cross_attention(fp32, 2, 8, 5, 1, 1, 64, 64, 1.0, repeated, view(kv), view(kv), out, stream=stream())
    own = torch.ones(2, 64, device="cuda")
    capi.cross_attention(fp32, 2, 8, 5, 1, 1, 64, 64, 1.0, capi.View(own.data_ptr(), 64, 0, 64), view(kv), view(kv), out, stream=stream())
    assert (whole[:, 0] == 0).all() and (whole[:, 1:] - 1).abs().max() < 1e-6


def test_lengths_and_masks_that_an_output_or_the_workspace_would_overwrite_are_refused():
    fp32, b, n, m = PRECISION["fp32"], 2, 3, 5000
    q, k = torch.zeros(b, n, 1, 16, device="cuda"), torch.zeros(b, m, 1, 16, device="cuda")
    room = capi.cross_attention_workspace(fp32, b, n, m, 1, 1, 16, 16)
    assert room > 0
    out, space = torch.zeros(8 + b * n * 16, device="cuda")[8:].view(b, n, 1, 16), torch.zeros(room // 4, device="cuda")
    lengths, keys, rows = torch.full((b,), m, dtype=torch.int32, device="cuda"), torch.ones(b, m, device="cuda"), torch.ones(b, n, device="cuda")

    def call(**given):
        capi.cross_attention(fp32, b, n, m, 1, 1, 16, 16, 1.0, view(q), view(k), view(k), view(out), workspace=space.data_ptr(), workspace_bytes=room,
                             stream=stream(), **given)

    names = dict(q_lengths="the query lengths", k_lengths="the key lengths", key_mask="the key mask", query_mask="the query mask")
    for what, name in names.items():
        for into, who in ((out, "out"), (space, "the workspace")):
            with pytest.raises(capi.KBError, match=f"{who} overlaps {name}"):
                call(**{what: into.data_ptr() + 8})
    # the last element alone, behind the start of the output
    with pytest.raises(capi.KBError, match="out overlaps the key lengths"):
        call(k_lengths=out.data_ptr() - 4)
    call(k_lengths=lengths.data_ptr(), key_mask=keys.data_ptr(), query_mask=rows.data_ptr())
    torch.cuda.synchronize()


# ---- a wait that ran out ----

@pytest.mark.parametrize("op", ("matmul", "rope", "attention"))
def test_a_wait_that_ran_out_is_reported_by_the_next_call_of_any_operator(op):
    """The word that a kernel would leave its code in, set by hand: the next call says so and launches nothing, the one after is as ever."""
    word = getattr(capi.lib(), "_ZN2kb16operatorWaitWordEv")
    word.restype, word.argtypes = ctypes.c_void_p, []
    t = torch.ones(1, 4, 1, 8, device="cuda")
    pos, freqs = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.zeros(4, 1, device="cuda")

    def call():
        out = torch.zeros_like(t)
        if op == "matmul":
            multiply("fp32", t[0, :, 0], t[0, :, 0], y=out[0, :, 0, :4])
        elif op == "rope":
            capi.rope(PRECISION["fp32"], 1, 4, 8, 8, pos.data_ptr(), 0, 1, freqs.data_ptr(), 1, 0, view(t), view(out), 1, stream=stream())
        else:
            attend("fp32", t, t, t, out, 1.0)
        return out

    torch.cuda.synchronize()
    ctypes.c_int.from_address(word()).value = 301
    with pytest.raises(capi.KBError, match=r"wait timed out in an earlier operator call \(code 301\)"):
        call()
    assert call().abs().sum() > 0


# ---- matmul ----

@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m,n,k", [(3, 136, 72), (3, 65, 33), (12, 136, 4096), (40, 136, 2048), (300, 264, 72), (300, 65, 33), (3000, 1200, 64)])
def test_matmul_activations_of_infinities_and_nan(dtype, m, n, k):
    """relu, mish and silu of +infinity are +infinity, of NaN NaN: in the row that has it and nowhere else."""
    g = seeded(dtype, m, n, k)
    x, w, bias = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=k ** -0.5), normal(g, n)
    w[:, 5] = w[:, 5].abs() + 0.25
    x[1, 5], x[2, 7] = INF, NAN
    others = [i for i in range(m) if i not in (1, 2)]
    for act in (1, 2, 3, 12):
        y = multiply(dtype, x, w, bias, act)
        assert (y[1] == INF).all(), act
        assert y[2].isnan().all(), act
        assert torch.isfinite(y[others]).all(), act

@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m,k", [(1, 72), (3, 72), (20, 72), (20, 2048), (129, 40), (300, 72), (300, 2048), (700, 33), (3000, 136), (140, 2048)])
@pytest.mark.parametrize("n", (1, 3, 6, 33, 62, 100, 257, 1203))
def test_matmul_writes_its_columns_only(dtype, m, k, n):
    """Rows of y on 16-byte boundaries, an end of no whole vector: what lies behind it in the same sixteen bytes belongs to somebody else."""
    g = seeded(dtype, m, n, k)
    x, w = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=k ** -0.5)
    other = normal(g, m, n, dtype=dtype)
    ld = (n + 7) // 8 * 8 + 8
    for residual in ("none", "other", "itself"):
        whole = torch.full((m, ld), 7.0, dtype=TYPES[dtype], device="cuda")
        y = whole[:, :n]
        if residual == "itself":
            y.copy_(other)
        padded = torch.full((m, ld), NAN, dtype=TYPES[dtype], device="cuda")
        padded[:, :n] = other
        r = dict(none=None, other=padded[:, :n], itself=y)[residual]
        want, bound = matmul_reference(dtype, x, w, None, 0, None if r is None else r.clone())
        assert_within(multiply(dtype, x, w, None, 0, r, y), want, bound, residual)
        assert (whole[:, n:] == 7.0).all(), residual

def test_matmul_of_the_longest_sums():
    """Rows on odd boundaries, of the most channels that there may be: the sums take more than two seconds, which is no reason to give them up.
    All but a few products are zeros, so the result is exact."""
    m, k = 17, (1 << 30) - 1
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 2 * (m + 1) * k + (4 << 30):
        pytest.skip("not enough memory")
    x, w = torch.zeros(m, k, dtype=torch.float16, device="cuda"), torch.zeros(1, k, dtype=torch.float16, device="cuda")
    places = [0, k // 2, k - 1]
    for i, at in enumerate(places):
        x[:, at] = torch.arange(m, device="cuda") % 7 + i
        w[:, at] = 2 ** i
    want = x[:, places].double() @ w[:, places].double().t()
    y = multiply("fp16", x, w)
    torch.cuda.synchronize()
    assert torch.equal(y.double(), want)
    one = torch.ones(32, 32, dtype=torch.float16, device="cuda")
    assert (multiply("fp16", one, one) == 32).all()  # and no later call has anything to report
    del x, w
    torch.cuda.empty_cache()


# ---- rope ----

PI = Fraction(31415926535897932384626433832795028841971693993751058209749445923078164062862089986280348253421170679, 10 ** 100)


def assert_turned_exactly(q, got, positions, freqs):
    """Every pair (adjacent channels, one head) of q against its angle in whole numbers.  Bound: the angle is off by 2^-26 of a turn (9.4e-8) for
    its rounding to fp32 and 2^-32 for its lower bits, sine and cosine by two steps (1.2e-7), and there are three roundings of 2^-24
    (1.8e-7): 2^-21 (4.8e-7) of |x0| + |x1|, and 2^-24 of the result."""
    for t in range(q.shape[1]):
        for p in range(freqs.shape[1]):
            total = sum(Fraction(int(positions[0, t, a])) * Fraction(float(freqs[0, p, a])) for a in range(freqs.shape[2]))
            rest = float(total - math.floor(total / (2 * PI)) * 2 * PI)
            x0, x1 = (float(q[0, t, 0, 2 * p + i]) for i in (0, 1))
            for i, exact in ((0, x0 * math.cos(rest) - x1 * math.sin(rest)), (1, x0 * math.sin(rest) + x1 * math.cos(rest))):
                allowed = (abs(x0) + abs(x1)) * 2.0 ** -21 + 2.0 ** -24 * abs(exact)
                off = abs(float(got[0, t, 0, 2 * p + i]) - exact)
                assert off <= allowed, (int(positions[0, t, 0]), float(freqs[0, p, 0]), off, allowed)


@pytest.mark.parametrize("axes", (1, 3, 16))
def test_rope_at_the_farthest_positions(axes):
    """int32 positions to the last, frequencies of a quarter to half a turn: the angle is off by a fraction of an fp32 step of a turn there too,
    however many axes add up."""
    g = seeded(axes)
    n, pairs = 24, 64
    q = torch.zeros(1, n, 1, 2 * pairs, device="cuda")
    q[..., 0::4] = q[..., 3::4] = 1  # (1, 0) and (0, 1)
    positions = torch.randint(2 ** 30, 2 ** 31 - 1, (1, n, axes), generator=g, device="cuda").to(torch.int32)
    positions[0, ::2] *= -1
    positions[0, 0], positions[0, 1] = 2 ** 31 - 1, -2 ** 31
    freqs = 1.6 + 1.5 * torch.rand(1, pairs, axes, generator=g, device="cuda")
    got, _ = turn("fp32", q, None, positions, freqs, 2 * pairs, False)
    assert_turned_exactly(q.cpu(), got.cpu(), positions.cpu(), freqs.cpu())


def test_rope_of_large_frequencies():
    """Many turns a step: what the two words of 1 / 2 pi say of a fraction of a turn is used to the last bit."""
    g = seeded("large")
    freqs = torch.tensor([12345.678, 3e6, 1e9, 2.0 ** 40, 1e13, 4.5e15, 3e16, 1.1e17, 7e17], device="cuda").view(1, 9, 1)
    q = normal(g, 1, 40, 1, 18)
    positions = torch.arange(-20, 20, device="cuda", dtype=torch.int32).view(1, 40, 1).contiguous()
    got, _ = turn("fp32", q, None, positions, freqs, 18, False)
    assert_turned_exactly(q.cpu(), got.cpu(), positions.cpu(), freqs.cpu())


# ---- attention ----

# one kernel after the other: few rows, one row tile whose keys two warpgroups share, two row tiles a block, both head sizes; CUDA cores
SHAPES = [(1, 2, 2, 64), (3, 4, 2, 128), (40, 2, 2, 64), (40, 4, 2, 128), (300, 6, 6, 64), (300, 6, 6, 128), (20, 2, 2, 136), (2, 2, 2, 20)]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,h,hk,d", SHAPES)
@pytest.mark.parametrize("at", (0, 130))
def test_attention_of_infinite_scores(dtype, n, h, hk, d, at):
    """Sixteen sequences with an infinity at another key each.  A score of +infinity makes its rows NaN (infinity - infinity), whichever key
    it is; one of -infinity leaves its key out.  The other heads are as ever."""
    _, q, k, v = attention_inputs(dtype, 16, n, 200, h, hk, d, d, at)
    q[..., 0] = q[..., 0].abs() + 0.25
    want, bound = attention_reference(dtype, q, k, v, d ** -0.5)
    for sign in (1, -1):
        kk = k.clone()
        for i in range(16):
            kk[i, at + i, 0, 0] = sign * INF
        out = attend(dtype, q, kk, v, empty_out(q, v), d ** -0.5)
        first = h // hk
        if sign > 0:
            assert out[:, :, :first].isnan().all()
        else:
            mask = torch.ones(16, 200, device="cuda")
            mask[torch.arange(16), at + torch.arange(16)] = 0
            assert_within(out[:, :, :first], *(t[:, :, :first] for t in attention_reference(dtype, q, k, v, d ** -0.5, key_mask=mask)))
        assert_within(out[:, :, first:], want[:, :, first:], bound[:, :, first:])


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,h,hk,d", SHAPES)
@pytest.mark.parametrize("m", (300, 4000))
@pytest.mark.parametrize("bad", (NAN, INF))
def test_attention_nan_is_seen_where_all_other_tiles_are_left_out(dtype, n, h, hk, d, m, bad):
    """Keys of one tile only, one of them NaN (or a score of infinity): whoever has the other tiles has nothing to add."""
    _, q, k, v = attention_inputs(dtype, 2, n, m, h, hk, d, d)
    q[..., 0] = q[..., 0].abs() + 0.25
    mask = torch.zeros(2, m, device="cuda")
    mask[0, 3:100] = 1
    mask[1, 140:250] = 1
    k[0, 50, 0, 0] = k[1, 200, 0, 0] = bad
    out = attend(dtype, q, k, v, empty_out(q, v), d ** -0.5, key_mask=mask)
    assert out[:, :, :h // hk].isnan().all()
    assert torch.isfinite(out[:, :, h // hk:]).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,h,hk,d", SHAPES)
@pytest.mark.parametrize("size", (30.0, 2500.0, 3e3, 1e5, 3e7, 1e9))
def test_attention_of_equal_large_scores(dtype, n, h, hk, d, size):
    """All keys of a sequence are the same, so all scores are, however large: a row is the mean of the values.  Equal scores have equal errors, so the
    bound (operator_cases.py) is that of the probabilities without that of the scores; 7.5e-5 more for the short polynomial of bf16."""
    m = 300
    _, q, k, v = attention_inputs(dtype, 2, n, m, h, hk, d, d, size)
    root = math.sqrt(size)
    q[:] = q * 0.01
    q[..., 0] = root * (1 + 0.01 * torch.arange(n, device="cuda")[:, None] / n)
    k[:] = k[:, :1] * 0.01
    k[0, ..., 0], k[1, ..., 0] = root, -root
    want = v.double().mean(1, keepdim=True).expand(-1, n, -1, -1).repeat_interleave(h // hk, 2)
    a = v.double().abs().mean(1, keepdim=True).expand(-1, n, -1, -1).repeat_interleave(h // hk, 2)
    u = torch.finfo(TYPES[dtype]).eps / 2
    bound = a * 2 * ((u if dtype != "fp32" else 0) + 2.0 ** -19 + (7.5e-5 if dtype == "bf16" else 0) + (m + 8) * 2.0 ** -23)
    out = attend(dtype, q, k, v, empty_out(q, v), 1.0)
    assert_within(out, want, bound + u * (want.abs() + bound) + (2.0 ** -25 if dtype == "fp16" else 0))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,h,hk,d", SHAPES)
@pytest.mark.parametrize("at", (0, 130))
def test_attention_of_one_key_far_above_the_others(dtype, n, h, hk, d, at):
    """Finite inputs whose scores reach 10^9: a row is the value of its largest key, whichever of sixteen that is, in rows of every size.  Bound: the
    probability, which need not be a power of two, is rounded to 16 bits in the sum of the values but not in the total (u, and 2^-19 for the
    exponential, as in operator_cases.py), and the result is rounded."""
    _, q, k, v = attention_inputs(dtype, 16, n, 200, h, hk, d, d, at)
    q[:], k[:] = 0, 0
    q[..., 0] = 40000.0 * 2.0 ** -(torch.arange(n, device="cuda") % 8)[:, None]
    k[..., 0] = -30000.0 * torch.rand(16, 200, 1, generator=seeded(n, h, d, at), device="cuda")
    for i in range(16):
        k[i, at + i, :, 0] = 31000.0 + 100 * i
    want = torch.stack([v[i, at + i] for i in range(16)]).double()[:, None].expand(-1, n, -1, -1).repeat_interleave(h // hk, 2)
    out = attend(dtype, q, k, v, empty_out(q, v), 1.0)
    u = torch.finfo(TYPES[dtype]).eps / 2
    bound = 2 * ((u if dtype != "fp32" else 0) + 2.0 ** -19) * want.abs()
    assert_within(out, want, bound + u * (want.abs() + bound) + (2.0 ** -25 if dtype == "fp16" else 0))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,h,hk,d", SHAPES)
@pytest.mark.parametrize("m", (700, 4000))
@pytest.mark.parametrize("rising", (True, False))
def test_attention_scores_that_grow_into_the_thousands(dtype, n, h, hk, d, m, rising):
    """Small scores in some tiles of keys, thousands in others, with keys left out by masks and lengths in both, NaN and infinities in them."""
    g, q, k, v = attention_inputs(dtype, 2, n, m, h, hk, d, d, rising)
    steps = torch.linspace(0.05, 3000, m, device="cuda") if rising else torch.linspace(3000, 0.05, m, device="cuda")
    k[0] = (k[0].float() * steps[:, None, None]).to(k.dtype)
    k[1] = (k[1].float() * torch.where(torch.arange(m, device="cuda") < m // 2, 0.1, 2000.0)[:, None, None]).to(k.dtype)
    mask = (torch.rand(2, m, generator=g, device="cuda") < 0.7).float()
    mask[0, 128:260] = 0
    lengths = torch.tensor([m - 37, m], dtype=torch.int32, device="cuda")
    want, bound = attention_reference(dtype, q, k, v, 0.25, k_lengths=lengths, key_mask=mask)
    left_out = (torch.arange(m, device="cuda") >= lengths[:, None]) | (mask == 0)
    k[left_out], v[left_out] = NAN, INF
    out = attend(dtype, q, k, v, empty_out(q, v), 0.25, k_lengths=lengths, key_mask=mask)
    assert_within(out, want, bound)
    # whatever the scores' own rounding does to the weights, a row lies between its values
    kept = torch.where(left_out[..., None, None], 0, v).double().abs().amax(1, keepdim=True).repeat_interleave(h // hk, 2)
    assert (out.double().abs() <= kept * 1.01).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,h,hk,d", SHAPES)
@pytest.mark.parametrize("gap", (12.0, 17.95, 23.5))
@pytest.mark.parametrize("m,every,at", [(8192, 8192, 0), (8192, 8192, 8191), (2000, 16, 0), (2000, 16, 15)])
def test_attention_small_weights_that_add_up(dtype, n, h, hk, d, gap, m, every, at):
    """Keys that take most of the weight (one, or one of every sixteen) and have values of 0, and thousands whose weights are 2^-gap of
    theirs: what a row is, is their sum, so each of them has to be as good as the bound says (a rounding of u of itself, however small
    it is)."""
    _, q, k, v = attention_inputs(dtype, 2, n, m, h, hk, d, d, gap, every)
    q[:], k[:] = 0, 0
    q[..., 0] = 1
    k[..., 0] = -gap * math.log(2.0)
    v[:] = (v.abs() + 4) * 1024
    k[:, at::every] = 0
    v[:, at::every] = 0
    want, bound = attention_reference(dtype, q, k, v, 1.0)
    assert_within(attend(dtype, q, k, v, empty_out(q, v), 1.0), want, bound)

@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,h,hk,d", SHAPES)
def test_attention_of_tokens_that_hold_nothing_and_rows_of_minus_infinity(dtype, n, h, hk, d):
    """What a masked token and one behind the last hold (NaN, infinities) reaches no other row; a row all of whose scores are -infinity has no
    key left, and is zeros."""
    _, q, k, v = attention_inputs(dtype, 3, n, 300, h, hk, d, d)
    tokens = torch.tensor([n, max(1, n // 2), n], dtype=torch.int32, device="cuda")
    live = (torch.arange(n, device="cuda") % 3 != 1).float().expand(3, n).contiguous()
    want, bound = attention_reference(dtype, q, k, v, 0.125, query_mask=live)
    nothing = torch.tensor([NAN, INF, -INF, 60000.0], device="cuda")[torch.arange(n, device="cuda") % 4].to(q.dtype)[None, :, None, None]
    dead = (live == 0) | (torch.arange(n, device="cuda") >= tokens[:, None])
    q = torch.where(dead[..., None, None], nothing, q)
    out = torch.full_like(empty_out(q, v), 7.0)
    attend(dtype, q, k, v, out, 0.125, q_lengths=tokens, query_mask=live)
    for i in range(3):
        rows = int(tokens[i])
        assert_within(out[i, :rows].flatten(0, 1), want[i, :rows].flatten(0, 1), bound[i, :rows].flatten(0, 1))
        assert (out[i, rows:] == 7.0).all()
    q[:], k[0] = 1, -INF
    out = attend(dtype, q, k, v, empty_out(q, v), 0.125)
    assert (out[0] == 0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,h,hk,d", SHAPES)
@pytest.mark.parametrize("scale", (1e-45, 1e-30, 1e30))
def test_attention_of_tiny_and_huge_scales(dtype, n, h, hk, d, scale):
    """A scale of next to nothing makes a row the mean of its values; a huge one brings back scores that are next to nothing."""
    m = 300
    _, q, k, v = attention_inputs(dtype, 2, n, m, h, hk, d, d, scale)
    if scale < 1:
        want, bound = attention_reference(dtype, q * 0, k, v, 1.0)
    elif dtype == "fp16":
        return  # its products are never that small
    else:
        q, k = q * 1e-15, k * 1e-15
        want, bound = attention_reference(dtype, q, k, v, scale)
    assert_within(attend(dtype, q, k, v, empty_out(q, v), scale), want, bound)


# ---- threads ----

@pytest.mark.parametrize("op", ("matmul wide", "matmul few", "matmul skinny", "attention few", "attention", "attention fp32", "rope"))
def test_the_first_call_of_a_thread(op):
    """A thread that has not touched its device yet, with buffers that another one has made."""
    g = seeded(op)
    x, w = normal(g, 3000, 512, dtype="bf16"), normal(g, 256, 512, dtype="bf16", scale=0.05)
    rows = {"matmul wide": 3000, "matmul few": 3, "matmul skinny": 100}.get(op, 0)
    dtype = "fp32" if "fp32" in op else "fp16"
    q, kv = normal(g, 2, 3 if op == "attention few" else 40, 4, 64, dtype=dtype), normal(g, 2, 300, 4, 64, dtype=dtype)
    positions, freqs = torch.arange(80, device="cuda", dtype=torch.int32).view(2, 40, 1), torch.full((1, 32, 1), 0.1, device="cuda")
    y, out = torch.zeros(max(rows, 1), 256, dtype=torch.bfloat16, device="cuda"), torch.zeros_like(q)
    space = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")

    def call():
        if rows:
            capi.matmul(PRECISION["bf16"], rows, 256, 512, x.data_ptr(), 512, w.data_ptr(), 512, y.data_ptr(), 256)
        elif op == "rope":
            capi.rope(PRECISION[dtype], 2, 40, 64, 64, positions.data_ptr(), 40, 1, freqs.data_ptr(), 1, 0, view(q), view(out), 4)
        else:
            b, n, h, d = q.shape
            capi.cross_attention(PRECISION[dtype], b, n, 300, h, h, d, d, 0.125, view(q), view(kv), view(kv), view(out), workspace=space.data_ptr(),
                                 workspace_bytes=1 << 22)

    got = y if rows else out
    call()
    torch.cuda.synchronize()
    want = got.clone()
    got.zero_()
    torch.cuda.synchronize()
    errors = []

    def work():
        try:
            call()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert want.abs().sum() > 0 and torch.equal(got, want)


# ---- graphs ----

def test_a_capture_that_forks_and_joins():
    """Operators on two streams of one capture, behind and before each other and torch's own kernels, each with a workspace of its own."""
    g = seeded("fork")
    x, w = normal(g, 200, 512, dtype="fp16"), normal(g, 256, 512, dtype="fp16", scale=0.04)
    q, kv = normal(g, 2, 3, 4, 64, dtype="fp16"), normal(g, 2, 6000, 4, 64, dtype="fp16")
    side = torch.cuda.Stream()

    def work(forked):
        here = torch.cuda.current_stream()
        a = multiply("fp16", x, w)
        there = side if forked else here
        there.wait_stream(here)
        with torch.cuda.stream(there):
            b = attend("fp16", q, kv, kv, empty_out(q, kv), 0.125)
            c = a * 2
            d = multiply("fp16", c, w[:, :256], act=3)
        e = attend("fp16", q, kv, kv, empty_out(q, kv), 0.25)
        here.wait_stream(there)
        return a, b, c, d, e, multiply("fp16", d, w[:, 256:], residual=a)

    want = [t.clone() for t in work(False)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(True)
    for _ in range(20):
        for t in got:
            t.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


FIRST_CALL = """
import torch
from tests.operator_cases import *
from tests.test_gpu_operators import *
g = seeded(1)
x, w = normal(g, 200, 512, dtype="fp16"), normal(g, 256, 512, dtype="fp16")
f, q, kv = x[:5].float(), normal(g, 2, 40, 4, 64, dtype="bf16"), normal(g, 2, 300, 4, 64, dtype="bf16")
positions, freqs = angles_for(g, 2, 40, 2, 1, 32, 100)
def work():
    return multiply("fp16", x, w), multiply("fp32", f, f), attend("bf16", q, kv, kv, empty_out(q, kv), 0.125), turn("bf16", q, None, positions, freqs, 64, False)[0]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = work()
for t in got: t.zero_()
graph.replay()
for a, b in zip(got, work()):
    assert torch.equal(a, b) and a.abs().sum() > 0
print("captured")
"""


def test_the_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ---- nets on boards that only this attention takes ----

@pytest.mark.parametrize("precision,tolerance,floor,step", [(capi.PRECISION_FP32, 2e-4, 1.0, None), (capi.PRECISION_FP16, 0.03, 3.0, 2.0 ** -11), (capi.PRECISION_BF16, 0.2, 3.0, 2.0 ** -8)])
@pytest.mark.parametrize("ylen,xlen", [(22, 22), (19, 25), (37, 20)])
def test_attention_blocks_of_nets_on_large_boards(ylen, xlen, precision, tolerance, floor, step, oracle):
    """Attention blocks of all kinds, boards of several sizes in one buffer, in every type against the oracle: element by element within the
    reference's tolerance of a layer (cpp/tests/testnn.cpp:8-15, as for the other blocks), and on the whole within two steps of a 16-bit
    type.  (Eight roundings of a value, of weights, inputs, queries, keys, values, probabilities and results, each off by half a step at
    most and evenly spread, are sqrt(8 / 12) = 0.8 steps.)"""
    import numpy as np

    from katago_b200 import modelfile as mf
    from tests.test_gpu_parity import _attn_block
    g, rng = mf._Gen(78), np.random.default_rng(ylen * xlen)
    mask = np.zeros((3, ylen, xlen), np.float32)
    mask[0] = 1
    mask[1, :13, :xlen - 2] = 1
    mask[2, :ylen - 7, :9] = 1
    on = mask > 0.5
    for channels, layer in [(384, _attn_block(g, 384, 6, 6, 64, 64, "learnable")), (384, _attn_block(g, 384, 6, 2, 64, 64, "fixed")),
                            (96, _attn_block(g, 96, 6, 3, 32, 16, "fixed")), (256, _attn_block(g, 256, 2, 2, 128, 128, "none"))]:
        x = rng.standard_normal((3, ylen, xlen, channels)).astype(np.float32) * mask[..., None]
        blob = mf.layer_blob(layer)
        ref = oracle.eval_layer(blob, x, mask, channels)
        out = capi.eval_layer(blob, x, mask, channels, precision=precision)
        assert np.isfinite(out).all() and (out[~on] == 0).all()
        assert np.all(np.abs(out - ref) <= tolerance * np.maximum(np.maximum(np.abs(out), np.abs(ref)), floor)), (channels, np.abs(out - ref).max())
        if step:
            off = np.sqrt(np.mean((out - ref)[on] ** 2) / np.mean(ref[on] ** 2))
            assert off <= 2 * step, (channels, off / step)
