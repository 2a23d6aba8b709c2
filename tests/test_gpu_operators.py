"""kb_matmul, kb_rope and kb_cross_attention on the GPU against their definitions in 64 bits (bounds: operator_cases.py)."""
import math
import threading
import zlib
from fractions import Fraction

import pytest

torch = pytest.importorskip("torch")

from katago_b200 import capi  # noqa: E402
from tests.operator_cases import (PRECISION, TYPES, assert_within, attend, attention_reference, laid_out, matmul_reference,  # noqa: E402
                                  rope_reference, stream, view)

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

ALL = ("fp32", "fp16", "bf16")
NAN = float("nan")


def normal(gen, *shape, dtype="fp32", scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(TYPES[dtype])


def seeded(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


# ---- matmul ----

def multiply(dtype, x, w, bias=None, act=0, residual=None, y=None):
    (m, k), n = x.shape, w.shape[0]
    if y is None:
        y = torch.full((m, n), NAN, dtype=x.dtype, device="cuda")
    capi.matmul(PRECISION[dtype], m, n, k, x.data_ptr(), x.stride(0) if m > 1 else max(k, x.stride(0)), w.data_ptr(), w.stride(0) if n > 1 else max(k, w.stride(0)),
                y.data_ptr(), y.stride(0) if m > 1 else max(n, y.stride(0)), bias=0 if bias is None else bias.data_ptr(), act=act,
                residual=0 if residual is None else residual.data_ptr(), ldr=0 if residual is None else max(n, residual.stride(0)), stream=stream())
    return y


MATMULS = [
    # m, n, k: single tokens, tiles that end anywhere, widths that are no whole vector, one of everything
    (1, 1, 1), (1, 64, 64), (1, 4096, 384), (2, 7, 1000), (3, 129, 72), (4, 512, 4096), (5, 50, 33), (8, 257, 136), (9, 64, 64), (16, 256, 128),
    (17, 40, 24), (31, 1000, 520), (64, 384, 384), (65, 96, 200), (127, 128, 64), (128, 256, 512), (129, 130, 131), (300, 8, 1536), (361, 384, 1024),
    (700, 1152, 384), (1083, 362, 361), (1500, 512, 65), (40, 2048, 2048), (2048, 264, 264),
    # several tiles per SM, the last ones partial in both directions; K cut over a cluster with rows of x in two tiles
    (5000, 1000, 200), (20000, 136, 72), (2100, 2000, 40), (2100, 2001, 33), (200, 300, 2600),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m,n,k", MATMULS)
def test_matmul_against_its_definition(dtype, m, n, k):
    g = seeded(dtype, m, n, k)
    x, w = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=k ** -0.5)
    bias, residual = normal(g, n), normal(g, m, n, dtype=dtype)
    for act, b, r in ((0, None, None), (2, bias, residual), (3, bias, None), (1, None, residual)):
        want, bound = matmul_reference(dtype, x, w, b, act, r)
        assert_within(multiply(dtype, x, w, b, act, r), want, bound, f"act {act}")


# fp32 sums that blocks of a cluster share (K in 1, 2, 4 and 8 parts, the last one shorter), rows on and off 16-byte boundaries,
# tiles of each size with partial last ones, rows that are just too many for the kernel of few
SHARED_SUMS = [(20, 64, 8000), (17, 35, 8193), (100, 100, 2500), (200, 132, 4100), (361, 513, 1030), (361, 512, 4096), (64, 388, 260), (1000, 1000, 900),
               (1003, 1000, 2500), (1083, 364, 361), (2048, 700, 1100), (4001, 1201, 67), (4000, 1200, 33), (9, 4096, 4096), (16, 301, 2049), (12, 3001, 136), (17, 3001, 136)]


@pytest.mark.parametrize("m,n,k", SHARED_SUMS)
def test_matmul_shared_sums(m, n, k):
    g = seeded(m, n, k)
    x, w = normal(g, m, k, dtype="fp32"), normal(g, n, k, dtype="fp32", scale=k ** -0.5)
    bias, residual = normal(g, n), normal(g, m, n, dtype="fp32")
    want, bound = matmul_reference("fp32", x, w, bias, 2, residual)
    y = residual.clone()
    assert_within(multiply("fp32", x, w, bias, 2, y, y), want, bound, "adding to its own output")
    assert torch.equal(multiply("fp32", x, w, bias, 2, residual), y), "the same sums every time"
    want, bound = matmul_reference("fp32", x, w, None, 0, None)
    wide = torch.full((m, n + 5), 7.0, device="cuda")  # rows of y off 16-byte boundaries, the columns behind them untouched
    assert_within(multiply("fp32", x, w, y=wide[:, 1:1 + n]), want, bound, "rows in a wider buffer")
    assert (wide[:, 0] == 7).all() and (wide[:, 1 + n:] == 7).all()


# 16-bit rows on 4-byte boundaries and on none, in wide tiles and in shared sums; odd sums in rows of even length
@pytest.mark.parametrize("dtype", ("fp16", "bf16"))
@pytest.mark.parametrize("off", (0, 1, 2))
@pytest.mark.parametrize("m,n,k", [(278, 308, 4706), (135, 102, 1442), (10, 16, 678), (16, 181, 236), (34, 204, 46), (541, 1213, 1268), (4001, 300, 391), (129, 70, 517), (128, 129, 130)])
def test_matmul_rows_off_vectors(dtype, m, n, k, off):
    g = seeded(dtype, m, n, k, off)
    ld = (k + 1) // 2 * 2 + (2 if off < 2 else 3)
    x, w = (torch.full((rows, ld), NAN, dtype=TYPES[dtype], device="cuda")[:, off:off + k] for rows in (m, n))
    x.copy_(normal(g, m, k, dtype=dtype)), w.copy_(normal(g, n, k, dtype=dtype, scale=k ** -0.5))
    bias, residual = normal(g, n), normal(g, m, n, dtype=dtype)
    want, bound = matmul_reference(dtype, x, w, bias, 1, residual)
    got = multiply(dtype, x, w, bias, 1, residual)
    assert_within(got, want, bound)
    assert torch.equal(multiply(dtype, x, w, bias, 1, residual), got), "the same sums every time"


@pytest.mark.parametrize("dtype", ALL)
def test_matmul_every_activation(dtype):
    g = seeded(dtype)
    x, w, bias = normal(g, 50, 32, dtype=dtype, scale=4), normal(g, 48, 32, dtype=dtype), normal(g, 48, scale=10)
    for act in (0, 1, 2, 3, 12):
        want, bound = matmul_reference(dtype, x, w, bias, act, None)
        assert_within(multiply(dtype, x, w, bias, act), want, bound, f"act {act}")


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m", (3, 24, 200))
@pytest.mark.parametrize("shift", (0, 1, 8))
def test_matmul_rows_in_wider_buffers(dtype, m, shift):
    """Rows further apart than they are long, beginning at any element; what lies between them stays, and is not read."""
    n, k = 104, 88
    g = seeded(dtype, m, shift)
    pad = 24 if shift != 1 else 5
    whole = {}
    for name, rows, cols in (("x", m, k), ("w", n, k), ("r", m, n), ("y", m, n)):
        whole[name] = torch.full((rows, cols + pad), NAN, dtype=TYPES[dtype], device="cuda")
    x, w, r, y = (whole[i][:, shift:shift + c] for i, c in (("x", k), ("w", k), ("r", n), ("y", n)))
    x.copy_(normal(g, m, k, dtype=dtype)), w.copy_(normal(g, n, k, dtype=dtype)), r.copy_(normal(g, m, n, dtype=dtype))
    bias = normal(g, n)
    multiply(dtype, x, w, bias, 3, r, y)
    want, bound = matmul_reference(dtype, x, w, bias, 3, r)
    assert_within(y, want, bound)
    assert whole["y"][:, :shift].isnan().all() and whole["y"][:, shift + n:].isnan().all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m", (1, 5, 30, 200, 3000))
@pytest.mark.parametrize("n,k", [(70, 33), (130, 85), (264, 1301)])
def test_matmul_odd_sums_in_aligned_rows(dtype, m, n, k):
    """Rows on 16-byte boundaries whose last vector is cut: what lies behind it (NaN) is not summed."""
    g = seeded(dtype, m, n, k)
    ld = (k + 7) // 8 * 8 + 16
    x, w = (torch.full((rows, ld), NAN, dtype=TYPES[dtype], device="cuda")[:, 8:8 + k] for rows in (m, n))
    x.copy_(normal(g, m, k, dtype=dtype)), w.copy_(normal(g, n, k, dtype=dtype, scale=k ** -0.5))
    want, bound = matmul_reference(dtype, x, w, None, 3, None)
    assert_within(multiply(dtype, x, w, None, 3), want, bound)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m,n,k", [(4, 200, 96), (40, 96, 512), (600, 512, 128), (33, 17, 9)])
def test_matmul_adds_to_its_own_output(dtype, m, n, k):
    g = seeded(dtype, m, n)
    x, w, y = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype), normal(g, m, n, dtype=dtype)
    want, bound = matmul_reference(dtype, x, w, None, 0, y)
    multiply(dtype, x, w, None, 0, y, y)
    assert_within(y, want, bound)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m", (2, 20, 300))
def test_matmul_infinities_and_nan_stay_in_their_rows_and_columns(dtype, m):
    n, k = 136, 72
    g = seeded(dtype, m)
    x, w = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype)
    want, bound = matmul_reference(dtype, x, w, None, 0, None)
    x[1, 5], w[7, 3] = NAN, float("inf")
    y = multiply(dtype, x, w)
    rows, cols = [i for i in range(m) if i != 1], [j for j in range(n) if j != 7]
    assert y[1].isnan().all() and not torch.isfinite(y[:, 7]).any()
    assert_within(y[rows][:, cols], want[rows][:, cols], bound[rows][:, cols])


def test_matmul_of_no_rows_does_nothing():
    w = torch.ones(8, 8, device="cuda")
    capi.matmul(PRECISION["fp32"], 0, 8, 8, 0, 8, w.data_ptr(), 8, 0, 8, stream=stream())


# ---- rope ----

def turn(dtype, q, k, positions, freqs, rot, halves, in_place=False):
    b, n, _, d = q.shape if q is not None else k.shape
    shared = positions.shape[0] == 1 and b > 1
    args = []
    outs = []
    for x in (q, k):
        if x is None:
            args += [None, None, 0]
            outs.append(None)
            continue
        y = x if in_place else torch.full_like(x, NAN)
        args += [view(x), view(y), x.shape[2]]
        outs.append(y)
    capi.rope(PRECISION[dtype], b, n, d, rot, positions.data_ptr(), 0 if shared else n * positions.shape[2], positions.shape[2],
              freqs.data_ptr(), freqs.shape[0], int(halves), *args, stream=stream())
    return outs


ROPES = [
    # b, n, q heads, k heads, dim, rot, axes, tables
    (1, 1, 1, 1, 2, 2, 1, 1), (1, 1, 6, 6, 64, 64, 2, 1), (3, 1, 32, 8, 128, 128, 1, 1), (2, 361, 6, 2, 64, 64, 2, 2), (2, 30, 8, 4, 128, 64, 3, 4),
    (1, 77, 5, 5, 80, 48, 3, 1), (5, 13, 3, 1, 24, 10, 2, 1), (2, 9, 4, 0, 32, 32, 1, 1), (2, 9, 0, 4, 32, 32, 4, 2), (1, 1000, 1, 1, 256, 256, 3, 1),
    (70, 3, 2, 2, 18, 18, 1, 1),
]


def angles_for(g, b, n, axes, tables, pairs, far):
    positions = torch.randint(-far if far < 1 << 20 else 0, far, (b, n, axes), generator=g, device="cuda").to(torch.int32)
    freqs = (torch.rand(tables, pairs, axes, generator=g, device="cuda") * 10 - 9).exp()
    return positions, freqs


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("halves", (False, True))
@pytest.mark.parametrize("b,n,hq,hk,d,rot,axes,tables", ROPES)
def test_rope_against_its_definition(dtype, halves, b, n, hq, hk, d, rot, axes, tables):
    g = seeded(dtype, halves, b, n, hq, d)
    q, k = (normal(g, b, n, h, d, dtype=dtype) if h else None for h in (hq, hk))
    for rows, layout, in_place in ((b, "dense", False), (1, "wide", False), (b, "heads_first", True), (b, "odd", False)):
        positions, freqs = angles_for(g, rows, n, axes, tables, rot // 2, 5000)
        ins = [None if x is None else laid_out(x, layout) for x in (q, k)]
        wants = [None if x is None else rope_reference(dtype, x, positions, freqs, rot, halves) for x in (q, k)]
        for got, want in zip(turn(dtype, *ins, positions, freqs, rot, halves, in_place), wants):
            if want is not None:
                assert_within(got, *want, f"{layout}, in place {in_place}")


@pytest.mark.parametrize("dtype", ALL)
def test_rope_far_positions_are_as_good_as_near_ones(dtype):
    g = seeded(dtype)
    q = normal(g, 2, 40, 4, 64, dtype=dtype)
    positions, freqs = angles_for(g, 2, 40, 3, 1, 32, 1 << 30)
    positions[0, 0], positions[0, 1] = 2 ** 31 - 1, -2 ** 31
    want, bound = rope_reference(dtype, q, positions, freqs, 64, False)
    # the 64-bit reference's own angle: a sum of three products of up to 2^33, each off by 2^-53 of itself
    bound = bound + 2.0 ** -17 * q.double().abs().amax(-1, keepdim=True)
    got, _ = turn(dtype, q, None, positions, freqs, 64, False)
    assert_within(got, want, bound)
    # the same without that: the angle in whole numbers
    pi = Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)
    for t in (0, 1, 7):
        for p in (0, 13, 31):
            total = sum(Fraction(int(positions[0, t, a])) * Fraction(float(freqs[0, p, a])) for a in range(3))
            rest = float(total - math.floor(total / (2 * pi)) * 2 * pi)
            x0, x1 = (float(q[0, t, 0, 2 * p + i]) for i in (0, 1))
            exact = x0 * math.cos(rest) - x1 * math.sin(rest)
            allowed = (abs(x0) + abs(x1)) * 2.0 ** -20 + torch.finfo(TYPES[dtype]).eps / 2 * (abs(exact) + 2.0 ** -10)
            assert abs(float(got[0, t, 0, 2 * p]) - exact) <= allowed


def test_rope_in_place_on_a_merged_projection():
    """q and k are column ranges of one buffer whose other columns stay."""
    g = seeded(1)
    whole = normal(g, 2, 19, 3 * 4 * 32, dtype="fp16")
    before = whole.clone()
    q, k = whole[..., :128].unflatten(-1, (4, 32)), whole[..., 128:256].unflatten(-1, (4, 32))
    positions, freqs = angles_for(g, 2, 19, 2, 2, 16, 19)
    want = [rope_reference("fp16", before[..., i:i + 128].unflatten(-1, (4, 32)), positions, freqs, 32, False) for i in (0, 128)]
    turn("fp16", q, k, positions, freqs, 32, False, in_place=True)
    assert_within(q, *want[0])
    assert_within(k, *want[1])
    assert torch.equal(whole[..., 256:], before[..., 256:])


def test_rope_in_place_of_single_tokens_in_one_buffer():
    """The newest token of each sequence: q and k side by side, whatever stride the only token has."""
    g = seeded(2)
    whole = normal(g, 5, 3 * 64, dtype="bf16")
    before = whole.clone()
    positions, freqs = angles_for(g, 5, 1, 1, 1, 16, 1 << 20)
    q, k = (before[:, i:i + 64].reshape(5, 1, 2, 32) for i in (0, 64))
    want = [rope_reference("bf16", x, positions, freqs, 32, True) for x in (q, k)]
    v = [capi.View(whole.data_ptr() + 2 * 64 * i, 192, 0, 32) for i in (0, 1)]
    capi.rope(PRECISION["bf16"], 5, 1, 32, 32, positions.data_ptr(), 1, 1, freqs.data_ptr(), 1, 1, v[0], v[0], 2, v[1], v[1], 2, stream())
    for i in (0, 1):
        assert_within(whole[:, 64 * i:64 * i + 64].reshape(5, 1, 2, 32), *want[i])
    assert torch.equal(whole[:, 128:], before[:, 128:])


@pytest.mark.parametrize("tables", (64, 4096))
def test_rope_many_tables(tables):
    """More frequencies than a block keeps: they are converted where they are used."""
    g = seeded(tables)
    heads = tables
    q = normal(g, 1, 3, heads, 16, dtype="fp16")
    positions, freqs = angles_for(g, 1, 3, 9, tables, 8, 1000)
    freqs[1, 2, 4] = float("nan")
    got, _ = turn("fp16", q, None, positions, freqs, 16, True)
    want, bound = rope_reference("fp16", q, positions, freqs.nan_to_num(0.0), 16, True)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[:, :, 1, 2] = bad[:, :, 1, 10] = True
    assert got[bad].isnan().all()
    assert_within(torch.where(bad, 0, got), torch.where(bad, 0, want), bound)


def test_rope_of_an_infinite_frequency_is_nan_and_stays_in_its_pair():
    q = torch.ones(1, 3, 2, 8, device="cuda")
    positions = torch.arange(3, device="cuda", dtype=torch.int32).view(1, 3, 1).contiguous()
    freqs = torch.full((1, 4, 1), 0.5, device="cuda")
    freqs[0, 2, 0] = float("inf")
    got, _ = turn("fp32", q, None, positions, freqs, 8, False)
    assert got[..., 4:6].isnan().all() and torch.isfinite(got[..., [0, 1, 2, 3, 6, 7]]).all()


# ---- attention ----

ATTENTIONS = [
    # b, n, m, heads, kv heads, qk dim, v dim
    (1, 1, 1, 1, 1, 1, 1), (1, 1, 361, 6, 6, 64, 64), (2, 1, 1000, 8, 2, 128, 128), (3, 2, 777, 16, 2, 64, 64), (1, 1, 5000, 4, 1, 128, 128),
    (2, 5, 130, 12, 4, 96, 96), (1, 16, 2048, 8, 8, 64, 64), (2, 33, 65, 4, 2, 32, 16), (1, 100, 64, 6, 6, 64, 64), (2, 128, 128, 2, 2, 128, 128),
    (1, 361, 722, 6, 3, 64, 64), (2, 129, 257, 3, 1, 128, 64), (1, 300, 1000, 2, 2, 128, 128), (1, 200, 77, 5, 5, 40, 24), (1, 50, 60, 2, 1, 256, 256),
    (1, 70, 90, 2, 2, 37, 19), (4, 7, 513, 7, 1, 80, 80), (1, 1000, 31, 4, 4, 48, 64), (1, 3, 9000, 2, 2, 64, 128), (2, 60, 3000, 4, 2, 64, 64),
    (1, 20, 400, 20, 4, 128, 128), (1, 256, 512, 7, 7, 64, 64), (1, 64, 640, 6, 2, 72, 72),
]


def attention_inputs(dtype, b, n, m, h, hk, dq, dv, *key):
    g = seeded(dtype, b, n, m, h, dq, *key)
    return g, normal(g, b, n, h, dq, dtype=dtype), normal(g, b, m, hk, dq, dtype=dtype), normal(g, b, m, hk, dv, dtype=dtype)


def empty_out(q, v):
    return torch.full((q.shape[0], q.shape[1], q.shape[2], v.shape[3]), NAN, dtype=q.dtype, device="cuda")


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("b,n,m,h,hk,dq,dv", ATTENTIONS)
def test_attention_against_its_definition(dtype, b, n, m, h, hk, dq, dv):
    _, q, k, v = attention_inputs(dtype, b, n, m, h, hk, dq, dv)
    want, bound = attention_reference(dtype, q, k, v, dq ** -0.5)
    assert_within(attend(dtype, q, k, v, empty_out(q, v), dq ** -0.5), want, bound)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("b,n,m,h,hk,dq,dv", [(5, 1, 700, 8, 2, 64, 64), (5, 9, 300, 6, 6, 64, 64), (5, 150, 200, 4, 2, 128, 128), (5, 40, 333, 3, 3, 32, 16),
                                              (5, 129, 129, 2, 1, 48, 40), (6, 200, 500, 2, 2, 64, 64), (6, 2, 2000, 4, 2, 128, 128)])
@pytest.mark.parametrize("what", ("lengths", "mask", "both"))
def test_attention_left_out_keys_may_hold_anything(dtype, b, n, m, h, hk, dq, dv, what):
    """Sequences of no key, one key, some, all; masks that leave a sequence nothing, one key at a time, or a whole tile out.  What is
    left out holds NaN and infinities; rows without a key are zeros; rows behind the last token keep what they had."""
    g, q, k, v = attention_inputs(dtype, b, n, m, h, hk, dq, dv, what)
    lengths = torch.tensor([0, 1, m // 2 + 1, m, 63, 64][:b], dtype=torch.int32, device="cuda") if what != "mask" else None
    mask = None
    if what != "lengths":
        mask = (torch.rand(b, m, generator=g, device="cuda") < 0.5).float()
        mask[1] = 0
        mask[2, : m // 2] = 0
        mask[3] = 0
        mask[3, m - 1] = 2.5
        mask[4, :70] = 0
    valid = torch.ones(b, m, dtype=torch.bool, device="cuda")
    if lengths is not None:
        valid &= torch.arange(m, device="cuda") < lengths[:, None]
    if mask is not None:
        valid &= mask != 0
    for t, bad in ((k, (NAN, float("inf"))), (v, (float("-inf"), NAN))):
        t[~valid] = torch.tensor(bad[0], dtype=t.dtype, device="cuda")
        t[..., 1::2][~valid] = torch.tensor(bad[1], dtype=t.dtype, device="cuda")
    tokens = torch.tensor([n, n, max(0, n - 1), n, 0, n][:b], dtype=torch.int32, device="cuda")
    tokens_mask = (torch.rand(b, n, generator=g, device="cuda") < 0.8).float()
    want, bound = attention_reference(dtype, q, k, v, dq ** -0.5, k_lengths=lengths, key_mask=mask, query_mask=tokens_mask)
    out = torch.full_like(empty_out(q, v), 7.0)
    attend(dtype, q, k, v, out, dq ** -0.5, tokens, lengths, mask, tokens_mask)
    for i in range(b):
        rows = int(tokens[i])
        assert_within(out[i, :rows].flatten(0, 1), want[i, :rows].flatten(0, 1), bound[i, :rows].flatten(0, 1), f"sequence {i}")
        assert (out[i, rows:] == 7.0).all()
    dead = ~valid.any(1)
    for i in range(b):
        if dead[i]:
            assert (out[i, : int(tokens[i])] == 0).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("b,n,m,h,hk,dq,dv", [(40, 300, 130, 4, 4, 64, 64), (40, 300, 200, 12, 4, 128, 128), (75, 257, 129, 2, 2, 64, 40), (30, 260, 300, 10, 5, 96, 128),
                                              (150, 1, 900, 4, 2, 64, 64), (150, 20, 300, 2, 2, 64, 64)])
@pytest.mark.parametrize("ragged", (False, True))
def test_attention_with_more_blocks_than_sms(dtype, ragged, b, n, m, h, hk, dq, dv):
    """Blocks of two row tiles, the last round's apart, sequences in the order of their lengths."""
    g, q, k, v = attention_inputs(dtype, b, n, m, h, hk, dq, dv, ragged)
    lengths = mask = tokens = None
    if ragged:
        lengths = torch.randint(0, m + 1, (b,), generator=g, device="cuda").to(torch.int32)
        lengths[:3] = torch.tensor([0, m, 1])
        mask = (torch.rand(b, m, generator=g, device="cuda") < 0.7).float()
        mask[5, :] = 0
        mask[6, :128] = 0
        tokens = torch.randint(0, n + 1, (b,), generator=g, device="cuda").to(torch.int32)
        tokens[0] = n
        left_out = (torch.arange(m, device="cuda") >= lengths[:, None]) | (mask == 0)
        k[left_out], v[left_out] = NAN, float("inf")
    want, bound = attention_reference(dtype, q, k, v, dq ** -0.5, k_lengths=lengths, key_mask=mask)
    out = torch.full_like(empty_out(q, v), 7.0)
    attend(dtype, q, k, v, out, dq ** -0.5, tokens, lengths, mask)
    if tokens is not None:
        behind = torch.arange(n, device="cuda") >= tokens[:, None]
        assert (out[behind] == 7.0).all()
        out[behind], want[behind], bound[behind] = 0, 0, 0
    assert_within(out.flatten(0, 1), want.flatten(0, 1), bound.flatten(0, 1))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ("heads_first", "wide", "odd"))
@pytest.mark.parametrize("n,m,h,hk,d", [(1, 300, 8, 2, 64), (150, 200, 4, 4, 64), (20, 90, 4, 2, 128), (260, 140, 3, 1, 32)])
def test_attention_layouts(dtype, layout, n, m, h, hk, d):
    _, q, k, v = attention_inputs(dtype, 2, n, m, h, hk, d, d, layout)
    want, bound = attention_reference(dtype, q, k, v, d ** -0.5)
    out = laid_out(empty_out(q, v), layout)
    attend(dtype, *(laid_out(t, layout) for t in (q, k, v)), out, d ** -0.5)
    assert_within(out, want, bound)


# keys that end in each sixteenth of a tile, and rows of out on and off 16-byte boundaries behind inputs that are on them
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ("dense", "odd"))
@pytest.mark.parametrize("n,m", [(70, 5), (3, 16), (70, 17), (90, 33), (5, 40), (70, 49), (33, 64), (70, 65), (20, 100), (90, 113)])
def test_attention_short_keys(dtype, layout, n, m):
    g, q, k, v = attention_inputs(dtype, 3, n, m, 4, 2, 48, 64, layout)
    k_lengths = torch.tensor([m, max(m - 16, 1), 0], dtype=torch.int32, device="cuda")
    k[1, max(m - 16, 1):], v[1, max(m - 16, 1):] = NAN, float("inf")
    k[2], v[2] = NAN, NAN
    want, bound = attention_reference(dtype, q, k, v, 0.2, k_lengths=k_lengths)
    assert_within(attend(dtype, q, k, v, laid_out(empty_out(q, v), layout), 0.2, k_lengths=k_lengths), want, bound)


@pytest.mark.parametrize("dtype", ALL)
def test_attention_repeated_inputs(dtype):
    """Strides of 0: one set of keys for all sequences, one value row for all heads."""
    _, q, k, v = attention_inputs(dtype, 3, 130, 90, 4, 4, 64, 64)
    k, v = k[:1].expand(3, -1, -1, -1), v[:, :, :1].expand(-1, -1, 4, -1)
    want, bound = attention_reference(dtype, q, k, v, 0.125)
    assert_within(attend(dtype, q, k, v, empty_out(q, v), 0.125), want, bound)
    q1 = q[:, :1].contiguous()
    want, bound = attention_reference(dtype, q1, k, v, 0.125)
    assert_within(attend(dtype, q1, k, v, empty_out(q1, v), 0.125), want, bound)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", (1, 140))
def test_attention_lengths_outside_their_range_read_nothing_else(dtype, n):
    _, q, k, v = attention_inputs(dtype, 2, n, 100, 2, 2, 64, 64)
    bad = torch.tensor([-5, 1 << 30], dtype=torch.int32, device="cuda")
    good = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    want, bound = attention_reference(dtype, q, k, v, 0.125, k_lengths=good)
    assert_within(attend(dtype, q, k, v, empty_out(q, v), 0.125, k_lengths=bad), want, bound)
    out = torch.full_like(empty_out(q, v), 7.0)
    attend(dtype, q, k, v, out, 0.125, q_lengths=bad)
    assert (out[0] == 7.0).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", (1, 140))
def test_attention_without_keys_is_zeros(dtype, n):
    q = torch.ones(2, n, 4, 64, dtype=TYPES[dtype], device="cuda")
    k = torch.empty(2, 0, 2, 64, dtype=TYPES[dtype], device="cuda")
    assert (attend(dtype, q, k, k, empty_out(q, k), 1.0) == 0).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", (1, 130))
def test_attention_scores_far_apart(dtype, n):
    """Scores of hundreds, rising and falling over the keys: the running maximum moves in every tile, or never after the first."""
    _, q, k, v = attention_inputs(dtype, 2, n, 600, 2, 2, 64, 64)
    k[0] *= torch.linspace(0.1, 30, 600, device="cuda").to(k.dtype)[:, None, None]
    k[1] *= torch.linspace(30, 0.1, 600, device="cuda").to(k.dtype)[:, None, None]
    want, bound = attention_reference(dtype, q, k, v, 0.25)
    assert_within(attend(dtype, q, k, v, empty_out(q, v), 0.25), want, bound)


@pytest.mark.parametrize("n", (1, 8, 130))
def test_attention_nan_of_an_attended_key_is_seen(n):
    _, q, k, v = attention_inputs("bf16", 2, n, 200, 2, 2, 64, 64)
    k[0, 150, 0, 3] = NAN
    out = attend("bf16", q, k, v, empty_out(q, v), 0.125)
    assert out[0, :, 0].isnan().all() and torch.isfinite(out[0, :, 1]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("n", (1, 20, 130))
def test_attention_offsets_past_32_bits(n):
    """Rows of a long cache: the last ones lie more than 2^32 elements from the first."""
    m, step = 300, (1 << 32) // 290 // 8 * 8
    room = torch.empty(step * (m - 1) + 256, dtype=torch.float16, device="cuda")
    k = torch.as_strided(room, (1, m, 2, 64), (0, step, 64, 1), 0)
    v = torch.as_strided(room, (1, m, 2, 64), (0, step, 64, 1), 128)
    _, q, kk, vv = attention_inputs("fp16", 1, n, m, 4, 2, 64, 64)
    k.copy_(kk), v.copy_(vv)
    want, bound = attention_reference("fp16", q, kk, vv, 0.125)
    assert_within(attend("fp16", q, k, v, empty_out(q, v), 0.125), want, bound)


# ---- all of them ----

def one_pass(s, out):
    """What a block does for one group of tokens: project, turn, look at kept states, project with the residual, feed forward."""
    b, n, c = s["x"].shape
    h, hk, d, dt = 6, 2, 64, "fp16"
    rows = b * n
    capi.matmul(PRECISION[dt], rows, h * d, c, s["x"].data_ptr(), c, s["wq"].data_ptr(), c, out["q"].data_ptr(), h * d, stream=stream())
    if s["fill"]:
        states = s["states"]
        m = states.shape[1]
        capi.matmul(PRECISION[dt], b * m, 2 * hk * d, c, states.data_ptr(), c, s["wkv"].data_ptr(), c, s["kv"].data_ptr(), 2 * hk * d, stream=stream())
        k = s["kv"][..., :hk * d].unflatten(-1, (hk, d))
        turn(dt, None, k, s["k_places"], s["freqs"], d, False, in_place=True)
    q = out["q"].view(b, n, h, d)
    turn(dt, q, None, s["q_places"], s["freqs"], d, False, in_place=True)
    k, v = (s["kv"][..., i:i + hk * d].unflatten(-1, (hk, d)) for i in (0, hk * d))
    attend(dt, q, k, v, out["a"].view(b, n, h, d), d ** -0.5, k_lengths=s["lengths"], workspace=out.get("ws"))
    capi.matmul(PRECISION[dt], rows, c, h * d, out["a"].data_ptr(), h * d, s["wo"].data_ptr(), h * d, out["x1"].data_ptr(), c, residual=s["x"].data_ptr(), ldr=c, stream=stream())
    f = s["w1"].shape[0]
    capi.matmul(PRECISION[dt], rows, f, c, out["x1"].data_ptr(), c, s["w1"].data_ptr(), c, out["f"].data_ptr(), f, bias=s["b1"].data_ptr(), act=2, stream=stream())
    capi.matmul(PRECISION[dt], rows, c, f, out["f"].data_ptr(), f, s["w2"].data_ptr(), f, out["y"].data_ptr(), c, residual=out["x1"].data_ptr(), ldr=c, stream=stream())
    return out["y"]


def block_state(n, seed, b=2, m=400, c=384, f=1024):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(x=normal(g, b, n, c, dtype="fp16"), states=normal(g, b, m, c, dtype="fp16"), wq=normal(g, 384, c, dtype="fp16", scale=c ** -0.5),
             wkv=normal(g, 256, c, dtype="fp16", scale=c ** -0.5), wo=normal(g, c, 384, dtype="fp16", scale=0.05), w1=normal(g, f, c, dtype="fp16", scale=c ** -0.5),
             b1=normal(g, f, scale=0.1), w2=normal(g, c, f, dtype="fp16", scale=0.03), kv=torch.empty(b, m, 256, dtype=torch.float16, device="cuda"),
             lengths=torch.tensor([m, m // 3], dtype=torch.int32, device="cuda"), fill=True)
    s["freqs"] = (torch.rand(1, 32, 3, generator=g, device="cuda") * 6 - 6).exp()
    s["q_places"] = torch.randint(0, 400, (b, n, 3), generator=g, device="cuda").to(torch.int32)
    s["k_places"] = torch.randint(0, 400, (b, m, 3), generator=g, device="cuda").to(torch.int32)
    return s


def block_buffers(n, b=2, c=384, f=1024):
    half = dict(dtype=torch.float16, device="cuda")
    out = dict(q=torch.empty(b * n, 384, **half), a=torch.empty(b * n, 384, **half), x1=torch.empty(b * n, c, **half), f=torch.empty(b * n, f, **half),
               y=torch.empty(b, n, c, **half))
    room = capi.cross_attention_workspace(PRECISION["fp16"], b, n, 400, 6, 2, 64, 64)
    out["ws"] = torch.empty(max(room, 16), dtype=torch.uint8, device="cuda")
    return out


def block_reference(s, x, q_places):
    b, n, c = x.shape
    x = x.double()
    q = (x @ s["wq"].double().t()).unflatten(-1, (6, 64))
    kv = s["states"].double() @ s["wkv"].double().t()
    k, v = kv[..., :128].unflatten(-1, (2, 64)), kv[..., 128:].unflatten(-1, (2, 64))
    q = rope_reference("fp16", q, q_places, s["freqs"], 64, False)[0]
    k = rope_reference("fp16", k, s["k_places"], s["freqs"], 64, False)[0]
    a = attention_reference("fp16", q, k, v, 0.125, k_lengths=s["lengths"])[0].flatten(2)
    x1 = x + a @ s["wo"].double().t()
    f = x1 @ s["w1"].double().t() + s["b1"].double()
    f = f * torch.tanh(torch.nn.functional.softplus(f))
    return x1 + f @ s["w2"].double().t()


def test_a_block_over_states_then_token_by_token():
    """A whole block against 64 bits, then the same tokens one at a time over the kept keys and values."""
    s = block_state(37, 5)
    whole = one_pass(s, block_buffers(37)).clone()
    want = block_reference(s, s["x"], s["q_places"])
    # every stage stores fp16 (2^-11 of a value) and the last sums 1024 and 384 products of such values: well below 1 % of the result
    assert (whole.double() - want).norm() <= 0.005 * want.norm()
    buffers = block_buffers(1)
    for i in (0, 17, 36):
        step = dict(s, x=s["x"][:, i:i + 1].contiguous(), q_places=s["q_places"][:, i:i + 1].contiguous(), fill=False)
        got = one_pass(step, buffers)
        assert (got[:, 0].double() - want[:, i]).norm() <= 0.005 * want[:, i].norm()


@pytest.mark.parametrize("n", (1, 37, 150))
def test_a_block_captured_in_a_graph_and_on_another_stream(n):
    s, other = block_state(n, 6), block_state(n, 7)
    plain = one_pass(s, block_buffers(n)).clone()
    plain_other = one_pass(other, block_buffers(n)).clone()
    assert torch.equal(plain, one_pass(s, block_buffers(n)))  # the same bits again
    torch.cuda.synchronize()
    out = block_buffers(n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one_pass(s, out)
    out["y"].fill_(NAN)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out["y"], plain)
    for name in ("x", "states", "wq", "wkv", "wo", "w1", "w2", "b1", "q_places", "k_places", "freqs", "lengths"):
        s[name].copy_(other[name])  # new inputs in the same buffers
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out["y"], plain_other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = one_pass(other, block_buffers(n))
    side.synchronize()
    assert torch.equal(again, plain_other)


def test_blocks_from_several_threads_at_once():
    states = [block_state(n, 20 + n) for n in (1, 20, 140, 3)]
    want = [one_pass(s, block_buffers(s["x"].shape[1])).clone() for s in states]
    torch.cuda.synchronize()
    got, errors = [None] * len(states), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                out = block_buffers(states[i]["x"].shape[1])
                for _ in range(20):
                    y = one_pass(states[i], out)
                torch.cuda.current_stream().synchronize()
                got[i] = y
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(states))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ---- nets on boards that only this attention takes ----

@pytest.mark.parametrize("ylen,xlen", [(22, 22), (19, 25), (37, 20)])
def test_transformer_nets_on_large_boards(ylen, xlen, oracle):
    """Boards whose keys and values do not fit a block's shared memory (above about 19x19), against the oracle; a position's result does
    not depend on the batch that it is evaluated in."""
    import numpy as np

    from katago_b200 import modelfile as mf
    from tests.test_gpu_parity import _assert_fp32_close, _assert_reduced_close, _rect_positions
    sp, gl = _rect_positions(3, ylen, xlen, seed=ylen * 100 + xlen)
    mask = sp[..., 0].reshape(3, -1)
    for tree in (mf.make_transformer(seed=61, layers=2), mf.make_transformer(seed=9, layers=2, d=64, heads=2, head_dim=32, ffn=96, rope="fixed")):
        blob = mf.to_blob(tree)
        ref = oracle.OracleModel(blob, nn_x=xlen, nn_y=ylen).forward(sp, gl)
        for prec in (capi.PRECISION_FP32, capi.PRECISION_FP16, capi.PRECISION_BF16):
            h = capi.Handle(capi.Model(blob), 3, nn_x=xlen, nn_y=ylen, precision=prec)
            got = h.forward(sp, gl)
            one = h.forward(sp[1:2], gl[1:2])
            h.close()
            if prec == capi.PRECISION_FP32:
                _assert_fp32_close(got, ref, mask)
            elif prec == capi.PRECISION_FP16:
                _assert_reduced_close(got, ref, mask)
            for key in one:
                assert np.array_equal(one[key][0], got[key][1]), key


def test_a_large_board_with_a_relative_position_bias_is_refused():
    from katago_b200 import modelfile as mf
    with pytest.raises(capi.KBError, match="larger than the relative-position bias table|relative-position bias"):
        capi.Handle(capi.Model(mf.to_blob(mf.make_transformer_relbias(seed=62, layers=1))), 1, nn_x=22, nn_y=22, precision=capi.PRECISION_FP16)


# ---- refusals that need a device ----

def test_refusals_of_pointers_and_overlaps():
    a = torch.zeros(64, 64, device="cuda")
    host = torch.zeros(64, 64)
    fp32 = PRECISION["fp32"]

    def mm(x, w, y, residual=0, n=16, ldy=64):
        capi.matmul(fp32, 16, n, 16, x, 64, w, 64, y, ldy, residual=residual, ldr=64, stream=stream())

    p = a.data_ptr()
    with pytest.raises(capi.KBError, match="not device memory"):
        mm(host.data_ptr(), p, p + 4 * 4096)
    with pytest.raises(capi.KBError, match="NULL"):
        mm(p, 0, p)
    with pytest.raises(capi.KBError, match="not aligned"):
        mm(p + 2, p, p)
    with pytest.raises(capi.KBError, match="y overlaps x"):
        mm(p, p + 16 * 256, p + 4)
    with pytest.raises(capi.KBError, match="y overlaps w"):
        mm(p, p + 16 * 256, p + 16 * 256)
    with pytest.raises(capi.KBError, match="y overlaps the residual"):
        mm(p, p + 64, p + 128, residual=p + 128 + 4)
    mm(p, p + 64, p + 128, residual=p + 128)  # column ranges of one buffer, and the residual in place
    t = torch.zeros(1, 8, 2, 16, device="cuda")
    pos, freqs = torch.zeros(8, 1, dtype=torch.int32, device="cuda"), torch.zeros(8, 1, device="cuda")
    with pytest.raises(capi.KBError, match="q out overlaps k in"):
        capi.rope(fp32, 1, 8, 16, 16, pos.data_ptr(), 0, 1, freqs.data_ptr(), 1, 0, view(t), view(t), 2, view(t), view(torch.zeros_like(t)), 2, stream())
    with pytest.raises(capi.KBError, match="overlap one another"):
        bad = capi.View(t.data_ptr(), 256, 8, 16)
        capi.rope(fp32, 1, 8, 16, 16, pos.data_ptr(), 0, 1, freqs.data_ptr(), 1, 0, view(t), bad, 2, stream=stream())
    with pytest.raises(capi.KBError, match="out overlaps v"):
        capi.cross_attention(fp32, 1, 8, 8, 2, 2, 16, 16, 1.0, view(torch.zeros_like(t)), view(torch.zeros_like(t)), view(t), view(t), stream=stream())
    room = capi.cross_attention_workspace(fp32, 1, 1, 5000, 1, 1, 16, 16)
    assert room > 0
    q, k = torch.zeros(1, 1, 1, 16, device="cuda"), torch.zeros(1, 5000, 1, 16, device="cuda")
    space = torch.empty(room, dtype=torch.uint8, device="cuda")
    with pytest.raises(capi.KBError, match="the workspace has"):
        capi.cross_attention(fp32, 1, 1, 5000, 1, 1, 16, 16, 1.0, view(q), view(k), view(k), view(torch.empty_like(q)), workspace=space.data_ptr(),
                             workspace_bytes=room - 1, stream=stream())
    torch.cuda.synchronize()
