"""The block operators over packed rows (gdc_packed_attention, gdc_linear_residual,
gdc_gated_residual_norm) on the GPU through the C ABI against their definitions in float64.

Tolerances count roundings: ``u`` is half a step of the output type (eps / 2, relative), sums of
n fp32 products may be off by n * 2^-23 times the sum of their magnitudes in any order."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"fp16": (torch.float16, 2), "bf16": (torch.bfloat16, 5)}


def _lib():
    from gliner_decide_metal_b200._lib import lib
    return lib


def _check(st):
    assert st == 0, _lib().gdc_last_error().decode()


def _done():
    torch.cuda.synchronize()
    _check(_lib().gdc_kernels_check_errors())


def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _normal(seed, *shape, std=1.0, mean=0.0, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)


def _within(got, want, tol):
    """|got - want| <= tol elementwise; not finite exactly where the definition is not."""
    g = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    assert torch.equal(g[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    over = (g - want).abs()[fine] - tol.expand_as(want)[fine]
    assert over.numel() == 0 or over.max().item() <= 0, f"off by {over.max().item():.3g} beyond the tolerance"


# ------------------------------------------------------------------------------------ attention

def _workspace(batch, q_rows, k_rows, heads, kv_heads, dim, fill=0xA5):
    n = C.c_size_t()
    _check(_lib().gdc_packed_attention_workspace(batch, q_rows, k_rows, heads, kv_heads, dim, C.byref(n)))
    return torch.full((max(256, n.value),), fill, dtype=torch.uint8, device="cuda")


def attention(q, k, v, q_off, k_off, heads, kv_heads, causal, scale=None, out=None, ws=None, stream=None):
    dim = q.shape[1] // heads
    code = 2 if q.dtype == torch.float16 else 5
    if out is None:
        out = torch.full((q.shape[0], heads * dim), 7.0, dtype=q.dtype, device="cuda")
    batch = q_off.numel() - 1
    ws = _workspace(batch, q.shape[0], k.shape[0], heads, kv_heads, dim) if ws is None else ws
    scale = 1 / math.sqrt(dim) if scale is None else scale
    _check(_lib().gdc_packed_attention(code, q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                                       out.data_ptr(), out.stride(0), q_off.data_ptr(), _p(k_off), batch, q.shape[0], k.shape[0],
                                       heads, kv_heads, dim, int(causal), scale, ws.data_ptr(), ws.numel(),
                                       _stream() if stream is None else stream))
    return out


def attention_definition(q, k, v, q_off, k_off, heads, kv_heads, causal, scale, fill):
    """float64 result (rows outside every sequence = fill) and the tolerance of every value."""
    dim = q.shape[1] // heads
    u = torch.finfo(q.dtype).eps / 2
    want = fill.double().clone()
    tol = torch.zeros_like(want)
    qo, ko = q_off.tolist(), (q_off if k_off is None else k_off).tolist()
    for b in range(len(qo) - 1):
        lq, lk = qo[b + 1] - qo[b], ko[b + 1] - ko[b]
        if lq == 0:
            continue
        see = torch.ones(lq, lk, dtype=torch.bool, device="cuda")
        if causal:
            see = see.tril(lk - lq)
        for h in range(heads):
            hk = h // (heads // kv_heads)
            cols = slice(h * dim, (h + 1) * dim)
            kcols = slice(hk * dim, (hk + 1) * dim)
            qb = q[qo[b]:qo[b + 1], cols].double()
            kb, vb = k[ko[b]:ko[b + 1], kcols].double(), v[ko[b]:ko[b + 1], kcols].double()
            rows = slice(qo[b], qo[b + 1])
            if lk == 0:
                want[rows, cols] = 0
                continue
            s = (qb @ kb.t() * scale).masked_fill(~see, -math.inf)
            w = torch.softmax(s, -1)
            w = torch.where(see.any(1, keepdim=True), w, torch.zeros_like(w)).masked_fill(~see, 0.0)
            # a value no query of the sequence sees stays out: 0 * inf is not part of the sum
            o = torch.zeros(lq, dim, dtype=torch.float64, device="cuda")
            fin = torch.isfinite(vb).all(1)
            o += w[:, fin] @ vb[fin]
            for j in torch.nonzero(~fin).flatten().tolist():
                o += torch.where(see[:, j:j + 1], w[:, j:j + 1] * vb[j][None], torch.zeros_like(o))
            o = torch.where(torch.isnan(s.masked_fill(~see, 0.0)).any(1, keepdim=True), torch.full_like(o, math.nan), o)
            want[rows, cols] = o
            # a score is off by ds (fp32 sum of dim products, its product with log2 e, the exponent's
            # own rounding); a weight by the rounding of its 16-bit form u and 2^-13 of the exponential's
            # polynomial, and twice (numerator, denominator) by ds
            mag = (qb.abs() @ kb.abs().t() * scale).masked_fill(~see, 0.0).nan_to_num(0, 0, 0).amax(1, keepdim=True)
            ds = (dim + 8) * 2.0 ** -23 * mag
            reach = w.nan_to_num(0.0) @ vb.abs().nan_to_num(0, 0, 0)
            tol[rows, cols] = (u + 2.0 ** -13 + lk * 2.0 ** -23 + 2 * ds) * (reach + o.abs().nan_to_num(0, 0, 0)) * 1.01 \
                + u * o.abs().nan_to_num(0, 0, 0) + torch.finfo(q.dtype).smallest_normal * u
    return want, tol


def _offsets(lengths, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(lengths)]), dtype=torch.int32, device="cuda")


def _attention_case(seed, dtype, lq, lk, heads, kv_heads, dim, causal, first=0, behind=0, fused=False, scale=None, same=False):
    t = DTYPES[dtype][0]
    tq, tk = first + sum(lq) + behind, first + sum(lk) + behind
    if fused:
        x = _normal(seed, tk, (heads + 2 * kv_heads) * dim + 8, dtype=t)
        q, k, v = x[:, :heads * dim], x[:, heads * dim:(heads + kv_heads) * dim], x[:, (heads + kv_heads) * dim:-8]
    else:
        q, k, v = (_normal(seed + i, r, w * dim, dtype=t) for i, (r, w) in enumerate([(tq, heads), (tk, kv_heads), (tk, kv_heads)]))
    q_off = _offsets(lq, first)
    k_off = None if same else _offsets(lk, first)
    got = attention(q, k, v, q_off, k_off, heads, kv_heads, causal, scale)
    _done()
    sc = np.float32(1 / math.sqrt(dim) if scale is None else scale).item()
    want, tol = attention_definition(q, k, v, q_off, k_off, heads, kv_heads, causal, sc, torch.full_like(got, 7.0))
    _within(got, want, tol)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,heads,kv_heads", [
    ([1], 1, 1), ([2], 3, 1), ([127], 2, 2), ([128], 2, 1), ([129], 4, 4), ([255, 1, 0, 257], 4, 2), ([300, 5, 700], 8, 2),
    ([0, 0, 33], 5, 1), ([64] * 9, 16, 4), ([511], 12, 4), ([640], 7, 1)])
def test_attention_prompts(dtype, dim, causal, lengths, heads, kv_heads):
    _attention_case(1, dtype, lengths, lengths, heads, kv_heads, dim, causal, first=3, behind=5, same=True)


@pytest.mark.parametrize("dtype,dim", [("fp16", 64), ("bf16", 128)])
@pytest.mark.parametrize("lq,lk,heads,kv_heads,causal", [
    ([1, 1, 1], [1, 700, 129], 8, 2, True), ([1], [5000], 4, 1, True), ([1] * 40, list(range(1, 1001, 25)), 8, 8, True),
    ([3, 0, 17], [300, 40, 17], 6, 2, True), ([130, 1], [900, 0], 4, 2, True), ([40, 9], [16, 3], 4, 2, True),
    ([5, 6], [0, 200], 2, 1, False), ([7, 100], [3000, 64], 16, 1, False), ([1, 2], [4097, 8000], 128, 1, True),
    ([1], [20000], 32, 4, True), ([2, 300, 1], [6000, 6000, 12000], 2, 2, True)])
def test_attention_last_rows_of_longer_sequences(dtype, dim, lq, lk, heads, kv_heads, causal):
    """Fewer queries than keys (single tokens, continued prompts), more queries than keys (rows that
    see nothing give zeros), sequences without queries or keys."""
    _attention_case(2, dtype, lq, lk, heads, kv_heads, dim, causal, first=2, behind=3)


@pytest.mark.parametrize("dtype,dim", [("fp16", 64), ("bf16", 64), ("fp16", 128)])
def test_attention_column_blocks_of_one_projection(dtype, dim):
    _attention_case(3, dtype, [130, 77], [130, 77], 8, 2, dim, True, fused=True, same=True)


@pytest.mark.parametrize("scale", [1e-4, 0.7, 3.0])
def test_attention_scales(scale):
    """From nearly uniform weights to rows that one key decides: the running maximum moves by much."""
    _attention_case(4, "fp16", [400], [400], 2, 1, 64, True, scale=scale, same=True)


def test_attention_long_sequence():
    _attention_case(5, "bf16", [2500], [2500], 4, 1, 128, True, same=True)


def test_attention_growing_scores():
    """Keys grow along the sequence, so that every key tile raises the maximum of every row."""
    n, dim = 1000, 64
    q = _normal(6, n, dim).abs()
    k = (_normal(7, n, dim).abs() * torch.linspace(0.05, 3, n, device="cuda")[:, None]).half()
    v = _normal(8, n, dim)
    off = _offsets([n])
    for causal in (True, False):
        got = attention(q, k, v, off, None, 1, 1, causal)
        _done()
        want, tol = attention_definition(q, k, v, off, None, 1, 1, causal, 0.125, torch.full_like(got, 7.0))
        _within(got, want, tol)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows,n", [(1, 250), (1, 6000), (150, 2000)])
@pytest.mark.parametrize("gap", [8.0, 14.0, 17.0, 17.375, 20.0])
def test_attention_small_weights_beside_a_dominant_key_of_zeros(dim, rows, n, gap):
    """One key outweighs every other by e^gap and its value row is zero, so the small weights are all there is. fp16
    weights have 2^-11 of themselves, or 2^-32 of the largest one (half the smallest fp16 step, 2^-25, at
    weights that are computed 2^7 larger)."""
    q, k, v = torch.zeros(rows, dim).half().cuda(), torch.zeros(n, dim).half().cuda(), 32 + 32 * _normal(37, n, dim).abs().clamp(max=1)
    q[:, 0], k[0, 0], v[0] = 1.0, gap, 0.0
    got = attention(q, k, v, _offsets([rows]), _offsets([n]), 1, 1, False, 1.0)
    _done()
    s = q.double() @ k.double().t()
    w = torch.softmax(s, -1)
    want = w @ v.double()
    u, ds = 2.0 ** -11, (dim + 8) * 2.0 ** -23 * gap
    tol = 2.0 ** -32 * w.amax(1, keepdim=True) * v.double().sum(0) + 2 * (u + 2.0 ** -22 + n * 2.0 ** -23 + 2 * ds) * want + u * want
    _within(got, want, tol)


@pytest.mark.parametrize("dtype,dim", [("fp16", 64), ("fp16", 128), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 6000), (150, 400)])
@pytest.mark.parametrize("scale", [0.125, 0.875, 1.0])
def test_attention_scores_beyond_what_fp32_counts_in(dtype, dim, rows, n, scale):
    """Scores of 10^6 to 10^11 whose largest is one key's by far: the output is that key's value row. The reference in log2
    units is rounded by up to a quarter, so the key's weight, 2^that, need not be a power of two: it is off by
    u when it is rounded to 16 bits (the row's sum takes it unrounded), and the output once more by u."""
    t = DTYPES[dtype][0]
    v = _normal(38, n, dim, dtype=t)
    for size in (400.0, 1000.0, 10000.0, 20000.0, 30000.0):
        q, k = torch.full((rows, dim), size, dtype=t, device="cuda"), torch.full((n, dim), size / 2, dtype=t, device="cuda")
        k[n // 2] = size
        got = attention(q, k, v, _offsets([rows]), _offsets([n]), 1, 1, False, scale)
        _done()
        want = v[n // 2].double().expand(rows, dim)
        _within(got, want, 2.02 * torch.finfo(t).eps / 2 * want.abs())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [1, 3, 200])
def test_attention_growing_scores_of_a_sequences_last_rows(dim, rows):
    """The same where one query tile's key tiles are taken in turn by both row groups, and in split ranges."""
    heads, lk = 4, [1500, 100, 3000]
    lq = [min(rows, n) for n in lk]
    q = _normal(24, sum(lq), heads * dim).abs()
    k = (_normal(25, sum(lk), 2 * dim).abs() * torch.cat([torch.linspace(0.05, 2, n, device="cuda") for n in lk])[:, None]).half()
    v = _normal(26, sum(lk), 2 * dim)
    qo, ko = _offsets(lq), _offsets(lk)
    got = attention(q, k, v, qo, ko, heads, 2, True, 0.125)
    _done()
    want, tol = attention_definition(q, k, v, qo, ko, heads, 2, True, 0.125, torch.full_like(got, 7.0))
    _within(got, want, tol)


@pytest.mark.parametrize("dtype,dim", [("fp16", 64), ("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_prompts_and_tokens_in_one_batch(dtype, dim, causal):
    """Every SM takes items of one and of two query tiles, of one key tile and of many, in mixed order."""
    rng = np.random.Generator(np.random.PCG64(23))
    lk = rng.integers(1, 700, 90)
    lq = np.where(rng.random(90) < 0.5, 1, np.minimum(lk, rng.integers(1, 400, 90)))
    _attention_case(23, dtype, lq.tolist(), lk.tolist(), 8, 4, dim, causal, first=1, behind=2)


@pytest.mark.parametrize("dtype,dim", [("fp16", 64), ("bf16", 128)])
@pytest.mark.parametrize("rows", [1, 60])
def test_attention_keys_of_weight_zero_before_an_infinite_value(dtype, dim, rows):
    """A row that an infinite value reaches keeps its other columns, although its first keys score -inf (weight 0)."""
    n, t = 300, DTYPES[dtype][0]
    q, k, v = _normal(27, rows, dim, dtype=t).abs(), _normal(28, n, dim, dtype=t), _normal(29, n, dim, dtype=t)
    k[:40, 5] = -math.inf
    v[100, 7] = math.inf
    qo, ko = _offsets([rows]), _offsets([n])
    got = attention(q, k, v, qo, ko, 1, 1, True)
    _done()
    assert (got[:, 7] == math.inf).all()
    v[100, 7] = 0
    want, tol = attention_definition(q, k, v, qo, ko, 1, 1, True, np.float32(1 / math.sqrt(dim)).item(), torch.full_like(got, 7.0))
    cols = [c for c in range(dim) if c != 7]
    _within(got[:, cols], want[:, cols], tol[:, cols])


@pytest.mark.parametrize("dtype,dim", [("fp16", 64), ("bf16", 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_keeps_what_is_not_seen_out(dtype, dim, bad):
    """Infinite and NaN keys and values reach exactly the queries that see them."""
    t = DTYPES[dtype][0]
    lengths = [200, 70]
    q, k, v = (_normal(10 + i, 300, w * dim, dtype=t) for i, w in enumerate([4, 2, 2]))
    off = _offsets(lengths)
    k[150, :dim] = bad   # one key head, seen by queries 150.. of the first sequence
    v[90, dim:] = bad    # the other head's values, inside the first tile
    v[270:] = bad        # behind the last sequence
    k[270:] = bad
    got = attention(q, k, v, off, None, 4, 2, True)
    _done()
    want, tol = attention_definition(q, k, v, off, None, 4, 2, True, np.float32(1 / math.sqrt(dim)).item(), torch.full_like(got, 7.0))
    first = got[:150, :2 * dim]
    assert torch.isfinite(first).all() and torch.isfinite(got[:90]).all() and torch.isfinite(got[200:270]).all()
    for rows, cols in ((slice(0, 150), slice(0, 2 * dim)), (slice(0, 90), slice(0, 4 * dim)), (slice(200, 300), slice(0, 4 * dim))):
        _within(got[rows, cols], want[rows, cols], tol[rows, cols])
    assert not torch.isfinite(got[90:200, 2 * dim:]).any()
    if not math.isinf(bad):
        assert torch.isnan(got[150:200, :2 * dim]).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows,n,causal", [(1, 1, True), (1, 2, True), (1, 200, False), (1, 7000, True), (40, 300, True), (500, 500, True),
                                           (700, 900, False), (3, 4000, True)])
@pytest.mark.parametrize("scale", [0.125, 0.75])
def test_attention_counts_its_roundings(dtype, dim, rows, n, causal, scale):
    """Every rounding of the computation and no more: a weight's 16-bit form (u; in fp16 at least 2^-32 of the largest weight), the
    exponential's 2^-22, sums of n terms and a score's dim products in fp32, the exponent's own rounding, and the
    output's u."""
    t = DTYPES[dtype][0]
    q, k, v = (_normal(46 + i, r, dim, dtype=t) for i, r in enumerate((rows, n, n)))
    got = attention(q, k, v, _offsets([rows]), _offsets([n]), 1, 1, causal, scale)
    _done()
    see = torch.ones(rows, n, dtype=torch.bool, device="cuda")
    see = see.tril(n - rows) if causal else see
    w = torch.softmax((q.double() @ k.double().t() * scale).masked_fill(~see, -math.inf), -1)
    want, reach = w @ v.double(), w @ v.double().abs()
    mag = (q.double().abs() @ k.double().abs().t() * scale).masked_fill(~see, 0.0).amax(1, keepdim=True)
    u, ds = torch.finfo(t).eps / 2, (dim + 8) * 2.0 ** -23 * mag
    smallest = 2.0 ** -32 * w.amax(1, keepdim=True) * (see.double() @ v.double().abs()) if dtype == "fp16" else 0.0
    weights = (u + 2.0 ** -22 + n * 2.0 ** -23 + 2 * ds) * (reach + want.abs()) * (1 + 2 * u) + smallest
    _within(got, want, weights * (1 + u) + u * want.abs() + torch.finfo(t).smallest_normal * u)


def test_attention_infinite_value_behind_many_keys():
    """64 rows that see an infinite value among 600,000 keys are computed by their definition, 32 by each of two warps one
    after the other (about 3 s); the CTA's other warps wait for them and its further items are computed."""
    dim, n, rows = 64, 600_000, 256 * 1200
    q, k, v = _normal(39, rows, dim), _normal(40, n, dim), _normal(41, n, dim, std=0.5, mean=1.0)
    v[n - 64, 0] = math.inf
    got = attention(q, k, v, _offsets([rows]), _offsets([n]), 1, 1, True, 0.125)
    _done()
    assert (got[-64:, 0] == math.inf).all() and torch.isfinite(got[:-64]).all() and torch.isfinite(got[-64:, 1:]).all()
    at = torch.tensor([0, 1000, 150_000, rows - 300, rows - 65, *range(rows - 64, rows)], device="cuda")
    v[n - 64, 0] = 0
    seen = (at + n - rows + 1)[:, None] > torch.arange(n, device="cuda")
    w = torch.softmax((q[at].double() @ k.double().t() * 0.125).masked_fill(~seen, -math.inf), -1)
    want, reach = w @ v.double(), w @ v.double().abs()
    ds = (dim + 8) * 2.0 ** -23 * (q[at].double().abs() @ k.double().abs().t() * 0.125).amax(1, keepdim=True)
    tol = (2.0 ** -11 + 2.0 ** -22 + n * 2.0 ** -23 + 2 * ds) * (reach + want.abs()) + 2.0 ** -11 * want.abs()
    _within(got[at][:, 1:], want[:, 1:], tol[:, 1:])
    assert (got > 0.5).all() and (got[:-64] < 1.5).all()  # (a row that was left out is 7)


def test_attention_skips_and_reports_bad_offsets():
    """Offsets that decrease or leave the rows: that sequence is skipped and reported, the others
    are computed."""
    dim, heads = 64, 2
    q, k, v = (_normal(20 + i, 96, heads * dim) for i in range(3))
    good = torch.tensor([0, 32, 64], dtype=torch.int32, device="cuda")
    for q_off, k_off in ([0, 32, 97], [0, 32, 64]), ([0, 32, 64], [0, 32, 200]), ([0, 32, 20], [0, 32, 64]), ([0, 32, 64], [0, 32, -5]):
        qo, ko = (torch.tensor(o, dtype=torch.int32, device="cuda") for o in (q_off, k_off))
        got = attention(q, k, v, qo, ko, heads, heads, True)
        torch.cuda.synchronize()
        assert _lib().gdc_kernels_check_errors() == 3
        want, tol = attention_definition(q, k, v, good[:2], good[:2], heads, heads, True, 0.125, torch.full_like(got, 7.0))
        _within(got[:32], want[:32], tol[:32])
        assert (got[32:] == 7.0).all()
    _done()


def test_attention_same_bits_on_every_call_and_replay():
    """Deterministic, whatever the workspace holds; a captured call follows new contents, lengths too."""
    dim, heads, kv = 128, 8, 2
    lk = [3000, 1, 900, 450]
    q, k, v = (_normal(30 + i, r, w * dim, dtype=torch.bfloat16) for i, (r, w) in enumerate([(4, heads), (sum(lk), kv), (sum(lk), kv)]))
    qo, ko = _offsets([1] * 4), _offsets(lk)
    a = attention(q, k, v, qo, ko, heads, kv, True)
    ws = _workspace(4, 4, k.shape[0], heads, kv, dim, fill=0xFF)
    b = attention(q, k, v, qo, ko, heads, kv, True, ws=ws)
    _done()
    assert torch.equal(a, b)
    out = torch.full_like(a, 7.0)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        attention(q, k, v, qo, ko, heads, kv, True, out=out, ws=ws)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, a)
    lk2 = [100, 2000, 1, 2250]
    ko.copy_(_offsets(lk2))
    q.copy_(_normal(40, 4, heads * dim, dtype=torch.bfloat16))
    g.replay()
    _done()
    want, tol = attention_definition(q, k, v, qo, ko, heads, kv, True, np.float32(1 / math.sqrt(dim)).item(), torch.full_like(out, 7.0))
    _within(out, want, tol)


def test_attention_two_streams_at_once():
    dim, heads = 64, 4
    off = _offsets([700, 300])
    xs = [tuple(_normal(50 + 3 * n + i, 1000, heads * dim) for i in range(3)) for n in range(2)]
    alone = [attention(*x, off, None, heads, heads, True) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    wss = [_workspace(2, 1000, 1000, heads, heads, dim) for _ in xs]
    outs = [torch.empty_like(a) for a in alone]
    torch.cuda.synchronize()
    for _ in range(5):
        for x, s, ws, o in zip(xs, streams, wss, outs):
            attention(*x, off, None, heads, heads, True, out=o, ws=ws, stream=s.cuda_stream)
    _done()
    assert all(torch.equal(a, o) for a, o in zip(alone, outs))


@pytest.mark.parametrize("dtype,dim", [("fp16", 64), ("bf16", 128)])
def test_attention_output_pitch_and_alignment(dtype, dim):
    """Outputs and inputs at 16-byte but not 32-byte addresses, with pitches above the width; what lies between
    the rows stays."""
    t = DTYPES[dtype][0]
    heads, kv, lens = 4, 2, [150, 3]
    n = sum(lens)
    x = _normal(11, n * ((heads + 2 * kv) * dim + 24) + 8, dtype=t)[8:].view(n, -1)
    q, k, v = x[:, :heads * dim], x[:, heads * dim + 8:(heads + kv) * dim + 8], x[:, (heads + kv) * dim + 16:(heads + 2 * kv) * dim + 16]
    flat = torch.full((n * (heads * dim + 8) + 8,), 7.0, dtype=t, device="cuda")
    out = flat[8:].view(n, heads * dim + 8)[:, :heads * dim]
    off = _offsets(lens)
    attention(q, k, v, off, None, heads, kv, True, out=out)
    _done()
    want, tol = attention_definition(q, k, v, off, None, heads, kv, True, np.float32(1 / math.sqrt(dim)).item(), out)
    _within(out, want, tol)
    assert (flat[8:].view(n, -1)[:, heads * dim:] == 7.0).all() and (flat[:8] == 7.0).all()


def test_attention_without_any_keys():
    q = _normal(12, 40, 256)
    off = _offsets([33, 5], 1)
    out = torch.full_like(q, 7.0)
    ws = _workspace(2, 40, 0, 4, 4, 64)
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    _check(_lib().gdc_packed_attention(2, q.data_ptr(), 256, None, 0, None, 0, out.data_ptr(), 256, off.data_ptr(), zero.data_ptr(), 2, 40, 0,
                                       4, 4, 64, 1, 0.125, ws.data_ptr(), ws.numel(), _stream()))
    _done()
    assert (out[1:39] == 0).all() and (out[:1] == 7.0).all() and (out[39:] == 7.0).all()


def test_attention_rows_beyond_32_bit_offsets():
    """A key buffer of more than 2^31 elements: the last sequence lies behind that offset."""
    width, rows = 4096, 600_000
    kv = torch.zeros(rows, width, dtype=torch.float16, device="cuda")
    at = rows - 700
    kv[at:] = _normal(13, 700, width)
    k, v = kv[:, 1024:1024 + 128], kv[:, width - 128:]
    q = _normal(14, 3, 8 * 64)
    qo = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    ko = torch.tensor([at, at + 500, rows], dtype=torch.int32, device="cuda")
    got = attention(q, k, v, qo, ko, 8, 2, True)
    _done()
    want, tol = attention_definition(q, k, v, qo, ko, 8, 2, True, 0.125, torch.full_like(got, 7.0))
    _within(got, want, tol)


@pytest.mark.parametrize("batch,most", [(3000, 6), (700, 40), (40, 900)])
def test_attention_many_sequences(batch, most):
    rng = np.random.Generator(np.random.PCG64(batch))
    lk = rng.integers(0, most, batch)
    lq = np.minimum(lk, rng.integers(0, 3, batch))
    _attention_case(15, "fp16", lq.tolist(), lk.tolist(), 4, 2, 64, True)


@pytest.mark.parametrize("batch,longest,empty", [(1, 300, 0), (33, 1500, 3), (64, 300, 0), (128, 130, 70), (129, 130, 80)])
@pytest.mark.parametrize("dtype,dim", [("fp16", 64), ("bf16", 128)])
def test_attention_tokens_of_up_to_many_sequences(batch, longest, empty, dtype, dim):
    """Single tokens of batches around the sizes at which the calls are planned in another way, some without a query."""
    rng = np.random.Generator(np.random.PCG64(batch))
    lk = rng.integers(1, longest, batch)
    lk[0] = longest * 4
    lq = np.ones(batch, dtype=int)
    lq[rng.permutation(batch)[:empty]] = 0
    _attention_case(30, dtype, lq.tolist(), lk.tolist(), 8, 2, dim, True, first=0 if empty == 0 else 1, behind=0 if empty == 0 else 2)


@pytest.mark.parametrize("dtype,dim", [("fp16", 64), ("bf16", 128)])
@pytest.mark.parametrize("lk", [[130 + 97 * i for i in range(24)], [20] * 11 + [4000], [700] * 32, [1] * 20, [0] * 10 + [513] * 9])
def test_attention_tokens_of_many_key_heads(dtype, dim, lk):
    """Items of more than a round, or of uneven length: split ranges of every length, joined."""
    _attention_case(33, dtype, [1] * len(lk), lk, 16, 8, dim, True, behind=1)


@pytest.mark.parametrize("dim,batch", [(64, 5), (128, 14), (64, 40)])
def test_attention_tokens_replayed_with_new_lengths(dim, batch):
    """A captured call follows the lengths that the offsets hold when it is replayed, whatever it split before."""
    heads, kv_heads, rows = 16, 8, 9000
    q, k, v = (_normal(34 + i, r, w * dim) for i, (r, w) in enumerate([(batch, heads), (rows, kv_heads), (rows, kv_heads)]))
    rng = np.random.Generator(np.random.PCG64(dim + batch))
    cuts = [np.sort(rng.integers(0, rows, batch - 1)) for _ in range(3)]
    cuts.append(np.arange(1, batch))  # one sequence has nearly all the keys
    offs = [torch.tensor(np.concatenate([[0], c, [rows]]), dtype=torch.int32, device="cuda") for c in cuts]
    qo, ko = torch.arange(batch + 1, dtype=torch.int32, device="cuda"), offs[0].clone()
    ws, out = _workspace(batch, batch, rows, heads, kv_heads, dim), torch.empty_like(q)
    attention(q, k, v, qo, ko, heads, kv_heads, True, out=out, ws=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        attention(q, k, v, qo, ko, heads, kv_heads, True, out=out, ws=ws)
    for off in offs + offs[:1]:
        ko.copy_(off)
        out.fill_(7.0)
        g.replay()
        _done()
        sc = np.float32(1 / math.sqrt(dim)).item()
        want, tol = attention_definition(q, k, v, qo, off, heads, kv_heads, True, sc, torch.full_like(out, 7.0))
        _within(out, want, tol)


def test_attention_tokens_with_bad_offsets():
    """Few single tokens: a sequence of bad offsets is skipped and reported, the others are computed."""
    heads, kv_heads, dim = 8, 2, 64
    q, k, v = (_normal(31 + i, r, w * dim) for i, (r, w) in enumerate([(6, heads), (4000, kv_heads), (4000, kv_heads)]))
    qo = torch.arange(7, dtype=torch.int32, device="cuda")
    ko = torch.tensor([0, 1000, 900, 1500, 3000, 4100, 4000], dtype=torch.int32, device="cuda")
    got = attention(q, k, v, qo, ko, heads, kv_heads, True)
    torch.cuda.synchronize()
    assert _lib().gdc_kernels_check_errors() == 3
    for b in range(6):
        if b in (1, 4, 5):
            assert (got[b] == 7.0).all()
            continue
        one = slice(ko[b].item(), ko[b + 1].item())
        want, tol = attention_definition(q[b:b + 1], k[one], v[one], _offsets([1]), _offsets([one.stop - one.start]), heads, kv_heads,
                                         True, 0.125, torch.full_like(got[b:b + 1], 7.0))
        _within(got[b:b + 1], want, tol)


def test_attention_refused_overlap_writes_nothing_out_of_place():
    """Offsets that decrease and make later sequences overlap earlier ones: reported, rows outside every sequence
    stay as they were."""
    heads, dim, n = 8, 64, 512
    q, k, v = (_normal(16 + i, n + 64, heads * dim) for i in range(3))
    off = torch.tensor([0, n, 0, n, 0, n, 0, n], dtype=torch.int32, device="cuda")
    got = attention(q, k, v, off, None, heads, heads, True)
    torch.cuda.synchronize()
    assert _lib().gdc_kernels_check_errors() == 3
    assert (got[n:] == 7.0).all()


@pytest.mark.parametrize("heads,rows", [(1, 1 << 20), (128, 1 << 17)])
def test_attention_refuses_overlaps_whose_items_pass_32_bits(heads, rows):
    """Offsets 0, rows, 0, rows, ...: every other sequence overlaps all the others, 2^31 and 2^32 items in all (256
    and 2 query rows each). Reported, and nothing is computed."""
    per_item = 2 * (128 // heads)
    assert rows // 2 * (rows // per_item) == (1 << 31 if heads == 1 else 1 << 32)
    q, kv = torch.zeros(rows, heads * 64, dtype=torch.float16, device="cuda"), _normal(19, 64, 64)
    odd = torch.arange(rows + 1, dtype=torch.int32, device="cuda") % 2
    got = attention(q, kv, kv, odd * rows, odd * 64, heads, 1, True)
    torch.cuda.synchronize()
    assert _lib().gdc_kernels_check_errors() == 3
    assert (got == 7.0).all()
    _done()


def test_attention_shared_workspace_in_turn():
    """Two captured calls on one workspace, replayed one after the other, again and again."""
    dim, heads = 64, 4
    cases, ws = [], _workspace(2, 2000, 6000, heads, heads, dim)
    for n, (lq, lk) in enumerate((([900, 100], [900, 100]), ([1, 1], [5000, 700]))):
        q, k, v = (_normal(17 + 3 * n + i, r, heads * dim) for i, r in enumerate((sum(lq), sum(lk), sum(lk))))
        qo, ko = _offsets(lq), _offsets(lk)
        alone = attention(q, k, v, qo, ko, heads, heads, True)
        out = torch.empty_like(alone)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            attention(q, k, v, qo, ko, heads, heads, True, out=out, ws=ws)
        cases.append((g, alone, out, (q, k, v, qo, ko)))
    for _ in range(3):
        for g, _, out, _ in cases:
            out.fill_(7.0)
            g.replay()
    _done()
    assert all(torch.equal(alone, out) for _, alone, out, _ in cases)


# --------------------------------------------------------------------------------------- linear

def linear(a, w, bias, residual, act, out=None, rows_dev=None):
    code = 2 if a.dtype == torch.float16 else 5
    M, N, K = a.shape[0], w.shape[0], a.shape[1]
    out = torch.full((M, N), 7.0, dtype=a.dtype, device="cuda") if out is None else out
    _check(_lib().gdc_linear_residual(code, a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(0), _p(bias), _p(residual),
                                      0 if residual is None else residual.stride(0), out.data_ptr(), out.stride(0), M, _p(rows_dev),
                                      N, K, act, _stream()))
    return out


def linear_definition(a, w, bias, residual, act):
    u = torch.finfo(a.dtype).eps / 2
    ad, wd = a.double(), w.double()
    z = ad @ wd.t()
    dz = a.shape[1] * 2.0 ** -23 * (ad.abs() @ wd.abs().t())
    if bias is not None:
        z = z + bias.double()
    dz = dz + 2.0 ** -23 * z.abs()
    f = [lambda t: t, torch.nn.functional.gelu, torch.relu, torch.nn.functional.silu][act](z)
    # the activations' slopes are below 1.13; their own evaluation is held to 2^-20 of |z|
    d = 1.13 * dz + 2.0 ** -20 * z.abs()
    want = f if residual is None else f + residual.double()
    return want, (d + 2.0 ** -23 * want.abs()) * (1 + u) + u * want.abs() + torch.finfo(a.dtype).smallest_normal * u


def _pitched(t, pad):
    """The same matrix with a row pitch larger by `pad`, the gap filled with NaN."""
    x = torch.full((t.shape[0], t.shape[1] + pad), math.nan, dtype=t.dtype, device="cuda")
    x[:, :t.shape[1]] = t
    return x[:, :t.shape[1]]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,N,K,act,bias,residual", [
    (1, 1, 8, 0, True, True), (1, 1024, 1024, 0, True, True), (1, 4096, 1000, 3, False, False), (2, 17, 24, 1, True, False),
    (7, 100, 72, 2, True, True), (16, 1000, 4096, 3, True, True), (33, 520, 136, 1, False, True), (64, 2048, 512, 1, True, True),
    (127, 96, 264, 0, False, False), (128, 256, 64, 2, False, True), (129, 257, 320, 1, True, True), (200, 1024, 1024, 3, True, True),
    (256, 512, 256, 0, True, True), (257, 384, 1024, 1, True, False), (500, 8, 2048, 0, True, True), (777, 1000, 1336, 3, False, True),
    (1000, 1, 64, 0, True, True), (1030, 1160, 200, 1, True, True), (2049, 2056, 136, 2, True, True), (4885, 1024, 512, 0, True, True)])
def test_linear(dtype, M, N, K, act, bias, residual):
    t = DTYPES[dtype][0]
    a, w = _normal(60, M, K, dtype=t), _normal(61, N, K, std=1 / math.sqrt(K), dtype=t)
    b = _normal(62, N, std=0.5, dtype=t) if bias else None
    r = _normal(63, M, N, dtype=t) if residual else None
    got = linear(a, w, b, r, act)
    again = linear(a, w, b, r, act)
    _done()
    _within(got, *linear_definition(a, w, b, r, act))
    assert torch.equal(got, again)


@pytest.mark.parametrize("M,N,K", [(5, 100, 64), (5, 96, 1000), (300, 260, 72), (300, 264, 72), (1030, 1024, 256)])
def test_linear_pitches_and_alignment(M, N, K):
    """Row pitches above the width (the gaps hold NaN), a K that no tile divides, outputs and
    residuals at odd pitches and addresses."""
    t = torch.float16
    a = _pitched(_normal(64, M, K, dtype=t), 8 - K % 8 + 16)
    w = _pitched(_normal(65, N, K, std=1 / math.sqrt(K), dtype=t), 8 - K % 8 + 8)
    b = torch.cat([torch.zeros(1, device="cuda", dtype=t), _normal(66, N, dtype=t)])[1:]
    for pad, shift in ((0, 0), (8, 0), (3, 1)):
        r = _pitched(_normal(67, M, N, dtype=t), pad)
        flat = torch.full((M * (N + pad) + 16,), 7.0, dtype=t, device="cuda")
        out = flat[shift:shift + M * (N + pad)].view(M, N + pad)[:, :N]
        linear(a, w, b, r, 1, out=out)
        _done()
        _within(out, *linear_definition(a, w, b, r, 1))
        if pad:
            assert (flat[shift:shift + M * (N + pad)].view(M, N + pad)[:, N:] == 7.0).all()
        assert (flat[shift + M * (N + pad):] == 7.0).all()


@pytest.mark.parametrize("K", [1, 3, 7, 63, 65, 129])
def test_linear_widths_below_the_pitch(K):
    a, w = (_pitched(_normal(68 + i, n, K), 16 - K % 8) for i, n in enumerate((40, 72)))
    got = linear(a, w, None, None, 0)
    _done()
    _within(got, *linear_definition(a, w, None, None, 0))


@pytest.mark.parametrize("M,N,K", [(64, 1024, 256), (1000, 512, 256), (600, 77, 64)])
def test_linear_in_place_and_device_row_count(M, N, K):
    """residual = out, and only the first *rows_dev rows computed and written."""
    a, w, x = _normal(70, M, K), _normal(71, N, K, std=1 / math.sqrt(K)), _normal(72, M, N)
    want, tol = linear_definition(a, w, None, x, 3)
    for rows in (M + 5, M, M - 1, M // 2 + 1, 1, 0, -4):
        out = x.clone()
        linear(a, w, None, out, 3, out=out, rows_dev=torch.tensor([rows], dtype=torch.int32, device="cuda"))
        _done()
        n = max(0, min(rows, M))
        _within(out[:n], want[:n], tol[:n])
        assert torch.equal(out[n:], x[n:])


def test_linear_carries_infinities_and_nan():
    """A row that is not finite spoils its own outputs and no others."""
    a, w = _normal(73, 300, 128), _normal(74, 200, 128, std=0.1)
    a[17, 5] = math.nan
    a[200, 9] = math.inf
    r = _normal(75, 300, 200)
    for act in (0, 1, 2, 3):
        got = linear(a, w, None, r, act)
        _done()
        keep = torch.ones(300, dtype=torch.bool, device="cuda")
        keep[[17, 200]] = False
        want, tol = linear_definition(a[keep], w, None, r[keep], act)
        _within(got[keep], want, tol)
        assert torch.isnan(got[17]).all()


@pytest.mark.parametrize("M", [1, 2, 300])
def test_linear_gelu_of_far_negative_values_in_bf16(M):
    """bf16 holds GELU(-6) = -6e-9 and GELU(-13) = -8e-38 like any other value: relative to the result, half a step (2^-8) and
    2^-14 of the evaluation (the fit's 1e-6, an exponent of up to 126 in fp32: 126 * 2^-24 ln 2 = 5e-6 for each of its
    three roundings). The power of two is zero below 2^-126 and its factor at most 1.2: results below 2^-125 may be zero."""
    t = torch.bfloat16
    z = torch.linspace(-14, -4, 1601, device="cuda").to(t)
    a, w = torch.zeros(M, 8, dtype=t, device="cuda"), torch.zeros(z.numel(), 8, dtype=t, device="cuda")
    a[:, 0], w[:, 0] = 1.0, z
    got = linear(a, w, None, None, 1)
    _done()
    zd = z.double()
    want = (0.5 * zd * torch.special.erfc(-zd / math.sqrt(2))).expand(M, -1)
    for far in (-20.0, -1e10, -3e38):
        w[:, 0] = far
        assert (linear(a, w, None, None, 1) == 0).all()
    _within(got, want, (2.0 ** -8 + 2.0 ** -14) * want.abs() + 2.0 ** -125)


def test_linear_captured_and_replayed():
    a, w, x = _normal(76, 90, 512), _normal(77, 520, 512, std=0.05), _normal(78, 90, 520)
    rows = torch.tensor([90], dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    linear(a, w, None, x, 1, out=out, rows_dev=rows)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        linear(a, w, None, x, 1, out=out, rows_dev=rows)
    a.copy_(_normal(79, 90, 512))
    rows.fill_(41)
    out.fill_(7.0)
    g.replay()
    _done()
    want, tol = linear_definition(a, w, None, x, 1)
    _within(out[:41], want[:41], tol[:41])
    assert (out[41:] == 7.0).all()


@pytest.mark.parametrize("M", [300, 4000])
def test_linear_rows_beyond_32_bit_offsets(M):
    """Output rows further apart than 2^31 elements in all: the last ones lie behind that offset."""
    pitch = 2 ** 31 // M + 4096
    a, w, r = _normal(80, M, 64), _normal(81, 40, 64, std=0.2), _normal(82, M, 40)
    flat = torch.empty(M * pitch, dtype=torch.float16, device="cuda")
    out = flat.view(M, pitch)[:, :40]
    out.copy_(r)
    linear(a, w, None, out, 0, out=out)
    _done()
    _within(out, *linear_definition(a, w, None, r, 0))


@pytest.mark.parametrize("M,N,K,act", [(64, 4096, 4096, 3), (256, 1024, 4096, 1), (2048, 4096, 1024, 1), (4885, 1024, 4096, 0), (3000, 2050, 520, 2),
                                       (1, 8192, 8192, 0), (130, 130, 8192, 1)])
def test_linear_forms_of_large_calls(M, N, K, act):
    """Every form the choice of tiles comes to: split K, one round of wide tiles, several rounds."""
    t = torch.bfloat16
    a, w, b, r = _normal(83, M, K, dtype=t), _normal(84, N, K, std=1 / math.sqrt(K), dtype=t), _normal(85, N, dtype=t), _normal(86, M, N, dtype=t)
    got = linear(a, w, b, r, act)
    _done()
    _within(got, *linear_definition(a, w, b, r, act))


# ----------------------------------------------------------------------------------------- norm

KINDS = {"none": 0, "layer": 1, "rms": 2}


def norm(y, x, post, pw, pb, gate, index, scale, pre, nw, nb, eps, x_out=None, n_out=None, rows_dev=None):
    code = 2 if x.dtype == torch.float16 else 5
    rows, cols = x.shape
    x_out = torch.full((rows, cols), 7.0, dtype=x.dtype, device="cuda") if x_out is None else x_out
    if n_out is None and pre != "none":
        n_out = torch.full((rows, cols), 7.0, dtype=x.dtype, device="cuda")
    _check(_lib().gdc_gated_residual_norm(code, _p(y), 0 if y is None else y.stride(0), x.data_ptr(), x.stride(0), KINDS[post], _p(pw),
                                          _p(pb), _p(gate), 0 if gate is None else gate.shape[0], _p(index), scale, KINDS[pre], _p(nw),
                                          _p(nb), x_out.data_ptr(), x_out.stride(0), _p(n_out), 0 if n_out is None else n_out.stride(0),
                                          rows, _p(rows_dev), cols, eps, _stream()))
    return x_out, n_out


def norm_definition(y, x, post, pw, pb, gate, index, scale, pre, nw, nb, eps):
    """(x', n) in float64, each with its tolerance: f fp32 roundings of every term, the statistics'
    sums of cols terms in fp32, one rounding of the result."""
    u, f = torch.finfo(x.dtype).eps / 2, 2.0 ** -24
    tiny = torch.finfo(x.dtype).smallest_normal * u
    cols = x.shape[1]
    n_sum = 8 + cols / 32  # terms of the longest chain a sum goes through, beyond the rounding of each

    def normed(z, dz, kind, w, b):
        """N(z) and how far it may be for a z that is off by dz."""
        wd = 1.0 if w is None else w.double()
        bd = 0.0 if b is None else b.double()
        if kind == "none":
            return z, dz
        mean = z.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(z[:, :1])
        dm = (dz + n_sum * f * z.abs()).mean(-1, keepdim=True) if kind == "layer" else 0.0
        d = z - mean
        inv = torch.rsqrt(d.square().mean(-1, keepdim=True) + eps)
        dd = dz + dm + f * (z.abs() + mean.abs())
        # rsqrt's slope: relative error of inv is at most half the relative error of the mean square
        dq = (2 * d.abs() * dd + dd * dd).mean(-1, keepdim=True) * inv * inv + n_sum * f + 4 * f
        h = d * inv
        dh = dd * inv + h.abs() * (0.5 * dq + 4 * f)
        out = h * wd + bd
        wa = 1.0 if w is None else wd.abs()
        return out, dh * wa + 2 * f * (h.abs() * wa + (0.0 if b is None else bd.abs()))

    xd = x.double()
    if y is None:
        x1, dx = xd, torch.zeros_like(xd)
    else:
        z, dz = normed(y.double(), torch.zeros_like(xd), post, pw, pb)
        if gate is not None:
            g = gate.double() if index is None else gate.double()[index.long()]
            z, dz = z * g, dz * g.abs() + f * (z * g).abs()
        x1 = xd + scale * z
        dx = abs(scale) * dz + 2 * f * (xd.abs() + abs(scale) * z.abs())
    outs = [(x1, dx * (1 + u) + u * x1.abs() + tiny)]
    if pre != "none":
        n, dn = normed(x1, dx, pre, nw, nb)
        outs.append((n, dn * (1 + u) + u * n.abs() + tiny))
    return outs


def _norm_inputs(seed, rows, cols, post, pre, gates, dtype, mean=0.0):
    t = DTYPES[dtype][0]
    y, x = _normal(seed, rows, cols, std=2.0, mean=mean, dtype=t), _normal(seed + 1, rows, cols, std=3.0, mean=mean, dtype=t)
    vec = lambda i, m: _normal(seed + i, cols, std=0.2, mean=m, dtype=t)  # noqa: E731
    pw, pb = (vec(2, 1.0), vec(3, 0.0)) if post != "none" else (None, None)
    nw, nb = (vec(4, 1.0), vec(5, 0.0)) if pre != "none" else (None, None)
    gate = _normal(seed + 6, gates, cols, dtype=t) if gates else None
    return y, x, pw, pb if post == "layer" else None, gate, nw, nb if pre == "layer" else None


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("post,pre", [("layer", "layer"), ("rms", "rms"), ("none", "layer"), ("rms", "none"), ("layer", "rms")])
@pytest.mark.parametrize("rows,cols,gate", [
    (1, 1, "none"), (1, 1024, "column"), (3, 7, "token"), (5, 64, "sequence"), (9, 257, "column"), (2, 1000, "none"),
    (33, 1024, "sequence"), (300, 768, "token"), (4, 2050, "column"), (7, 4096, "none"), (3, 8192, "sequence"), (2, 16384, "token"),
    (2, 16383, "column")])
def test_norm(dtype, post, pre, rows, cols, gate):
    gates = {"none": 0, "column": 1, "sequence": 3, "token": rows}[gate]
    y, x, pw, pb, g, nw, nb = _norm_inputs(80, rows, cols, post, pre, gates, dtype)
    index = torch.arange(rows, dtype=torch.int32, device="cuda") * 7 % 3 if gate == "sequence" else None
    args = (y, x, post, pw, pb, g, index, 0.5, pre, nw, nb, 1e-5)
    got = norm(*args)
    _done()
    for o, (want, tol) in zip(got, norm_definition(*args)):
        _within(o, want, tol)


@pytest.mark.parametrize("cols", [1024, 1000, 999])
def test_norm_rows_far_from_zero(cols):
    """A mean a hundred times the deviation: the statistics lose nothing."""
    y, x, pw, pb, g, nw, nb = _norm_inputs(90, 20, cols, "layer", "layer", 1, "fp16", mean=200.0)
    args = (y, x, "layer", pw, pb, g, None, 1.0, "layer", nw, nb, 1e-7)
    got = norm(*args)
    _done()
    for o, (want, tol) in zip(got, norm_definition(*args)):
        _within(o, want, tol)


def test_norm_constant_and_zero_rows():
    x = torch.zeros(4, 512, dtype=torch.float16, device="cuda")
    y = torch.full((4, 512), 3.0, dtype=torch.float16, device="cuda")
    w, b = _normal(92, 512, mean=1.0), _normal(93, 512)
    for kind in ("layer", "rms"):
        args = (y, x, kind, w, b, None, None, 1.0, kind, w, b, 1e-6)
        got = norm(*args)
        _done()
        for o, (want, tol) in zip(got, norm_definition(*args)):
            _within(o, want, tol)


@pytest.mark.parametrize("cols", [768, 333])
def test_norm_before_the_first_block_in_place_and_pitches(cols):
    """y NULL; x_out = x and n_out = y; row pitches above the width; rows behind *rows_dev."""
    y, x, pw, pb, g, nw, nb = _norm_inputs(94, 50, cols, "rms", "layer", 1, "bf16")
    args = (None, x, "none", None, None, None, None, 1.0, "layer", nw, nb, 1e-6)
    got = norm(*args)
    _done()
    assert torch.equal(got[0], x)
    _within(got[1], *norm_definition(*args)[1])

    x_out, y_out = x.clone(), y.clone()
    full = (y, x, "rms", pw, None, g, None, 0.25, "layer", nw, nb, 1e-6)
    want = norm_definition(*full)
    norm(y_out, x_out, *full[2:], x_out=x_out, n_out=y_out, rows_dev=torch.tensor([37], dtype=torch.int32, device="cuda"))
    _done()
    for o, (wt, tol), before in zip((x_out, y_out), want, (x, y)):
        _within(o[:37], wt[:37], tol[:37])
        assert torch.equal(o[37:], before[37:])

    wide = [torch.full((50, cols + 5), 7.0, dtype=x.dtype, device="cuda") for _ in range(2)]
    norm(_pitched(y, 3), _pitched(x, 8), *full[2:], x_out=wide[0][:, :cols], n_out=wide[1][:, :cols])
    _done()
    for o, (wt, tol) in zip(wide, want):
        _within(o[:, :cols], wt, tol)
        assert (o[:, cols:] == 7.0).all()


def test_norm_skips_and_reports_bad_gate_indices():
    y, x, pw, pb, g, nw, nb = _norm_inputs(96, 12, 256, "rms", "rms", 4, "fp16")
    index = torch.tensor([0, 1, 2, 3, 4, -1, 3, 2, 1, 0, 1 << 30, 2], dtype=torch.int32, device="cuda")
    ok = torch.tensor([0, 1, 2, 3, 6, 7, 8, 9, 11], device="cuda")
    got = norm(y, x, "rms", pw, None, g, index, 1.0, "rms", nw, None, 1e-6)
    torch.cuda.synchronize()
    assert _lib().gdc_kernels_check_errors() == 3
    want = norm_definition(y[ok], x[ok], "rms", pw, None, g, index[ok], 1.0, "rms", nw, None, 1e-6)
    for o, (wt, tol) in zip(got, want):
        _within(o[ok], wt, tol)
        assert (o[[4, 5, 10]] == 7.0).all()
    _done()


@pytest.mark.parametrize("pitch", [0, 3, -8, 1 << 40])
def test_pitches_of_absent_tensors_do_not_matter(pitch):
    lib = _lib()
    x, w, n = _normal(43, 8, 64), _normal(44, 64, 64, std=0.1), _normal(45, 8, 64)
    out, again, off, ws = torch.empty_like(x), torch.empty_like(x), _offsets([8]), _workspace(1, 8, 0, 1, 1, 64)
    args = (2, x.data_ptr(), 64, w.data_ptr(), 64, None, None)
    _check(lib.gdc_linear_residual(*args, pitch, out.data_ptr(), 64, 8, None, 64, 64, 0, _stream()))
    _check(lib.gdc_linear_residual(*args, 0, again.data_ptr(), 64, 8, None, 64, 64, 0, _stream()))
    _done()
    assert torch.equal(out, again)
    _check(lib.gdc_packed_attention(2, x.data_ptr(), 64, None, pitch, None, pitch, out.data_ptr(), 64, off.data_ptr(),
                                    torch.zeros_like(off).data_ptr(), 1, 8, 0, 1, 1, 64, 1, 0.125, ws.data_ptr(), ws.numel(), _stream()))
    _done()
    assert (out == 0).all()
    _check(lib.gdc_gated_residual_norm(2, None, pitch, x.data_ptr(), 64, 0, None, None, None, 0, None, 1.0, 2, None, None, None, pitch,
                                       out.data_ptr(), 64, 8, None, 64, 1e-6, _stream()))
    _check(lib.gdc_gated_residual_norm(2, n.data_ptr(), 64, x.data_ptr(), 64, 0, None, None, None, 0, None, 1.0, 0, None, None,
                                       again.data_ptr(), 64, None, pitch, 8, None, 64, 1e-6, _stream()))
    _done()
    _within(out, *norm_definition(None, x, "none", None, None, None, None, 1.0, "rms", None, None, 1e-6)[1])
    _within(again, *norm_definition(n, x, "none", None, None, None, None, 1.0, "none", None, None, 1e-6)[0])


def test_errors_of_several_calls_are_all_named():
    """The error word holds what every call since its last reading has raised: one status, and a message that names all."""
    lib = _lib()
    y, x, pw, pb, g, nw, nb = _norm_inputs(96, 12, 256, "rms", "rms", 4, "fp16")
    q = _normal(32, 8, 64)

    def bad_index():
        norm(y, x, "rms", pw, None, g, torch.full((12,), 4, dtype=torch.int32, device="cuda"), 1.0, "rms", nw, None, 1e-6)

    def bad_offsets():
        attention(q, q, q, torch.tensor([0, 9], dtype=torch.int32, device="cuda"), None, 1, 1, True)

    for raised, status in (((bad_index, bad_offsets), 3), ((bad_offsets, bad_index), 3), ((bad_offsets,), 3),
                           ((bad_index, lambda: _check(lib.gdc_selftest_wait_timeout(1000, _stream()))), 9)):
        for f in raised:
            f()
        torch.cuda.synchronize()
        assert lib.gdc_kernels_check_errors() == status
        message = lib.gdc_last_error().decode()
        assert ("gate index" in message) == (bad_index in raised) and ("packed offsets" in message) == (bad_offsets in raised)
        assert ("time limit" in message) == (status == 9)
        _done()


def test_norm_spoiled_row_stays_alone():
    y, x, pw, pb, g, nw, nb = _norm_inputs(97, 40, 640, "layer", "layer", 1, "fp16")
    y[7, 3], x[21, 600] = math.nan, math.inf
    args = (y, x, "layer", pw, pb, g, None, 1.0, "layer", nw, nb, 1e-6)
    got = norm(*args)
    _done()
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[7, 21]] = False
    want = norm_definition(y[keep], x[keep], *args[2:])
    for o, (wt, tol) in zip(got, want):
        _within(o[keep], wt, tol)
    assert torch.isnan(got[1][[7, 21]]).all()


@pytest.mark.parametrize("rows,cols", [(5000, 1024), (3000, 1001), (2500, 4096), (1500, 514), (700, 8200)])
def test_norm_many_rows_in_place(rows, cols):
    """More rows than the device holds at once, x and y overwritten row by row."""
    y, x, pw, pb, g, nw, nb = _norm_inputs(98, rows, cols, "layer", "rms", 7, "fp16")
    index = (torch.arange(rows, device="cuda") % 7).int()
    full = (y, x, "layer", pw, pb, g, index, 0.5, "rms", nw, None, 1e-6)
    want = norm_definition(*full)
    xo, no = x.clone(), y.clone()
    norm(no, xo, *full[2:], x_out=xo, n_out=no, rows_dev=torch.tensor([rows - 3], dtype=torch.int32, device="cuda"))
    _done()
    for o, (wt, tol), before in zip((xo, no), want, (x, y)):
        _within(o[:-3], wt[:-3], tol[:-3])
        assert torch.equal(o[-3:], before[-3:])


def test_norm_captured_and_replayed():
    y, x, pw, pb, g, nw, nb = _norm_inputs(99, 64, 384, "rms", "layer", 1, "bf16")
    rows = torch.tensor([64], dtype=torch.int32, device="cuda")
    args = (y, x, "rms", pw, None, g, None, 1.0, "layer", nw, nb, 1e-6)
    xo, no = norm(*args, rows_dev=rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm(*args, x_out=xo, n_out=no, rows_dev=rows)
    x.copy_(_normal(100, 64, 384, dtype=x.dtype))
    rows.fill_(50)
    xo.fill_(7.0), no.fill_(7.0)
    graph.replay()
    _done()
    for o, (wt, tol) in zip((xo, no), norm_definition(*args)):
        _within(o[:50], wt[:50], tol[:50])
        assert (o[50:] == 7.0).all()


# -------------------------------------------------------------------------------- a block of them

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_a_block_over_packed_rows(dtype):
    """Norm, fused projection, attention, output projection with residual, norm, FFN: one block over
    packed prompts with the row count on the device, each stage against its definition on the
    stage's own inputs, then captured once and replayed on shorter prompts."""
    t = DTYPES[dtype][0]
    cap, e, heads, kv, dim, ff = 700, 512, 8, 2, 64, 1024
    width = (heads + 2 * kv) * dim
    mk = lambda i, *s: _normal(100 + i, *s, std=1 / math.sqrt(s[-1]), dtype=t)  # noqa: E731
    wqkv, wo, w1, w2 = mk(0, width, e), mk(1, e, heads * dim), mk(2, ff, e), mk(3, e, ff)
    b1, n1, n2, post = _normal(110, ff, std=0.1, dtype=t), *(_normal(111 + i, e, std=0.1, mean=1.0, dtype=t) for i in range(3))
    x = _normal(115, cap, e, dtype=t)
    off = _offsets([300, 1, 211])
    rows = off[-1:]
    buf = lambda w: torch.full((cap, w), 7.0, dtype=t, device="cuda")  # noqa: E731
    h, qkv, ctx, y, x1, h2, mid, x2 = buf(e), buf(width), buf(heads * dim), buf(e), buf(e), buf(e), buf(ff), buf(e)
    ws = _workspace(3, cap, cap, heads, kv, dim)
    q, k, v = qkv[:, :heads * dim], qkv[:, heads * dim:(heads + kv) * dim], qkv[:, (heads + kv) * dim:]

    def block():
        norm(None, x, "none", None, None, None, None, 1.0, "rms", n1, None, 1e-6, x_out=x1, n_out=h, rows_dev=rows)
        linear(h, wqkv, None, None, 0, out=qkv, rows_dev=rows)
        attention(q, k, v, off, None, heads, kv, True, out=ctx, ws=ws)
        linear(ctx, wo, None, None, 0, out=y, rows_dev=rows)
        norm(y, x, "rms", post, None, None, None, 0.5, "rms", n2, None, 1e-6, x_out=x1, n_out=h2, rows_dev=rows)
        linear(h2, w1, b1, None, 3, out=mid, rows_dev=rows)
        linear(mid, w2, None, x1, 0, out=x2, rows_dev=rows)

    def verify():
        n = int(rows.item())
        _within(h[:n], *norm_definition(None, x[:n], "none", None, None, None, None, 1.0, "rms", n1, None, 1e-6)[1])
        _within(qkv[:n], *linear_definition(h[:n], wqkv, None, None, 0))
        want, tol = attention_definition(q, k, v, off, None, heads, kv, True, 0.125, torch.full_like(ctx, 7.0))
        _within(ctx, want, tol)
        _within(y[:n], *linear_definition(ctx[:n], wo, None, None, 0))
        for o, wt in zip((x1, h2), norm_definition(y[:n], x[:n], "rms", post, None, None, None, 0.5, "rms", n2, None, 1e-6)):
            _within(o[:n], *wt)
        _within(mid[:n], *linear_definition(h2[:n], w1, b1, None, 3))
        _within(x2[:n], *linear_definition(mid[:n], w2, None, x1[:n], 0))
        for o in (h, qkv, ctx, y, x1, h2, mid, x2):
            assert (o[n:] == 7.0).all()

    block()
    _done()
    verify()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        block()
    for o in (h, qkv, ctx, y, x1, h2, mid, x2):
        o.fill_(7.0)
    off.copy_(_offsets([5, 130, 260]))
    g.replay()
    _done()
    verify()


def test_calls_follow_each_other_without_waiting():
    """Kernels that start before the one ahead of them has ended still read its results: a long chain of
    dependent calls on one stream, each overwriting what the next reads, against the same chain with
    a wait after every call."""
    def chain(wait):
        x = _normal(200, 96, 512)
        w = [_normal(201 + i, 512, 512, std=0.04) for i in range(3)]
        off = _offsets([40, 56])
        ws = _workspace(2, 96, 96, 8, 8, 64)
        h, y, c = (torch.empty_like(x) for _ in range(3))
        for i in range(60):
            norm(None, x, "none", None, None, None, None, 1.0, "rms", None, None, 1e-6, x_out=y, n_out=h)
            wait()
            linear(h, w[i % 3], None, None, 0, out=y)
            wait()
            attention(y, h, y, off, None, 8, 8, True, out=c, ws=ws)
            wait()
            linear(c, w[(i + 1) % 3], None, x, 3, out=x)
            wait()
        torch.cuda.synchronize()
        return x
    a, b = chain(lambda: None), chain(torch.cuda.synchronize)
    _done()
    assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("cols", [512, 514, 515])
def test_norm_follows_a_gate_that_the_call_before_it_writes(cols):
    """Gate rows, weights and indices change between the calls of a chain: the gate and the weight are each written by the
    linear just before the norm that reads them. Against the same chain with a wait after every call."""
    def chain(wait):
        rows, gates = 700, 9
        x, y = _normal(210, rows, cols), _normal(211, rows, cols)
        c, w = _normal(212, 40, gates, 64), [_normal(213 + i, cols, 64, std=0.1) for i in range(3)]
        gate, weight = (torch.zeros(n, cols, dtype=torch.float16, device="cuda") for n in (gates, 1))
        index = (torch.arange(rows, device="cuda") % gates).int()
        for i in range(40):
            linear(c[i], w[i % 3], None, None, 0, out=gate)
            wait()
            norm(y, x, "rms", weight[0] if i else None, None, gate, index if i % 3 else index.roll(i), 0.5, "rms", None, None, 1e-6,
                 x_out=x, n_out=y)
            wait()
            linear(c[i][:1], w[(i + 1) % 3], None, None, 0, out=weight)
            wait()
        torch.cuda.synchronize()
        return x
    a, b = chain(lambda: None), chain(torch.cuda.synchronize)
    _done()
    assert torch.isfinite(a).all() and torch.equal(a, b)


def test_the_three_operators_on_streams_of_their_own():
    """Calls of every form at once on four streams, each against the same call alone."""
    w, a = _normal(220, 1024, 512, std=0.05), _normal(221, 900, 512)
    x, y, r = _normal(222, 900, 512), _normal(223, 900, 512), _normal(224, 900, 1024)
    q, kv, off = _normal(225, 900, 512), _normal(226, 900, 128), _offsets([500, 400])
    ws = _workspace(2, 900, 900, 8, 2, 64)
    calls = [lambda out: linear(a, w, None, r, 1, out=out), lambda out: linear(a[:5], w, None, r[:5], 3, out=out),
             lambda out: attention(q, kv, kv, off, None, 8, 2, True, out=out, ws=ws),
             lambda out: norm(y, x, "rms", None, None, None, None, 0.5, "layer", None, None, 1e-6, x_out=out[0], n_out=out[1])]
    make = lambda: [torch.empty_like(r), torch.empty_like(r[:5]), torch.empty_like(q), torch.empty(2, 900, 512, dtype=q.dtype, device="cuda")]  # noqa: E731
    alone, outs, streams = make(), make(), [torch.cuda.Stream() for _ in calls]
    for f, o in zip(calls, alone):
        f(o)
        torch.cuda.synchronize()
    for _ in range(20):
        for f, o, s in zip(calls, outs, streams):
            with torch.cuda.stream(s):
                f(o)
    _done()
    assert all(torch.equal(u, v) for u, v in zip(alone, outs))


def test_first_use_of_a_kernel_inside_a_capture():
    """Only the first call on a device has to come before a capture; a kernel first used inside one works."""
    import subprocess
    import sys
    code = """
import torch, sys
sys.path.insert(0, {root!r})
from tests import test_gpu_block_ops as t
t.linear(t._normal(1, 8, 64), t._normal(2, 16, 64), None, None, 0)
torch.cuda.synchronize()
q = t._normal(3, 400, 512, dtype=torch.bfloat16)
off = t._offsets([300, 100])
ws = t._workspace(2, 400, 400, 4, 4, 128)
outs = [torch.empty_like(q) for _ in range(3)]
w = t._normal(4, 512, 512, std=0.04, dtype=torch.bfloat16)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    t.attention(q, q, q, off, None, 4, 4, True, out=outs[0], ws=ws)
    t.linear(outs[0], w, None, q, 1, out=outs[1])
    t.norm(outs[1], q, "rms", None, None, None, None, 1.0, "layer", None, None, 1e-6, x_out=outs[2], n_out=outs[0])
g.replay()
t._done()
again = [torch.empty_like(q) for _ in range(3)]
t.attention(q, q, q, off, None, 4, 4, True, out=again[0], ws=ws)
t.linear(again[0], w, None, q, 1, out=again[1])
t.norm(again[1], q, "rms", None, None, None, None, 1.0, "layer", None, None, 1e-6, x_out=again[2], n_out=again[0])
t._done()
assert all(torch.equal(a, b) for a, b in zip(outs, again))
print("same")
"""
    from pathlib import Path
    root = str(Path(__file__).resolve().parents[1])
    r = subprocess.run([sys.executable, "-c", code.format(root=root)], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]
