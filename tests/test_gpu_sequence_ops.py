"""Sequence operators against plain float64 implementations.

Tolerances, per output, are sums of the roundings that the kernels document:
  * the output's own rounding, half a step of its type (BF16 2^-8, FP32 2^-24);
  * scores: products of FP32-class pieces (2^-20 of each) and an FP32 sum of d
    terms, together at most e_s = S (2^-20 + (d + 8) 2^-23) with S the sum of
    |products|; a weight then moves by e_s relative to its neighbours, twice
    after the normalisation;
  * weights: 2^-8 when rounded to BF16, 2^-11 to FP16, 2^-20 in two pieces, and
    2^-21 for the exponential;
  * the FP32 sum over n keys, (n + 8) 2^-23;
  all but the first relative to sum_j softmax_j |v_j|.
"""

import math

import numpy as np
import pytest

import ppocr_b200 as P

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def offsets(n):
    return torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device="cuda")


def attend(q, k, v, scale, first=None):
    """Float64 attention of one sequence: q [n, H, d], k / v [m, G, d]; query i sees keys 0 .. first + i (None:
    all).  Returns the output, sum softmax |v| and the largest sum of |products| of each row."""
    n, heads, d = q.shape
    m, kv = k.shape[:2]
    out, mag, prod = torch.zeros_like(q), torch.zeros_like(q), q.new_zeros(n, heads, 1)
    if n == 0 or m == 0:
        return out, mag, prod
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if first is not None:
        seen = torch.arange(m, device=q.device)[None] <= torch.arange(n, device=q.device)[:, None] + first
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        s = (q[:, h] @ kh.T * scale).masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        w = torch.where(seen, (s - torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp(), s.new_zeros(()))
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
        for i in range(n):   # masked values may hold anything: only seen ones are multiplied
            if not torch.isfinite(vh).all():
                c = int(seen[i].sum())
                out[i, h], mag[i, h] = w[i, :c] @ vh[:c], w[i, :c] @ vh[:c].abs()
        if torch.isfinite(vh).all():
            out[:, h], mag[:, h] = w @ vh, w @ vh.abs()
        prod[:, h] = torch.where(seen, (q[:, h].abs() @ kh.abs().T) * scale, s.new_zeros(())).amax(-1, keepdim=True)
    return out, mag, prod


def tolerance(ref, mag, prod, d, n, dtype, weight):
    e_s = prod * (2.0 ** -20 + (d + 8) * 2.0 ** -23)
    return HALF_STEP[dtype] * ref.abs() + mag * (weight + 2 * e_s + 2.0 ** -20 + (n + 8) * 2.0 ** -23) + 1e-30


def check(got, ref, tol, what=""):
    got = got.double()
    assert torch.isfinite(got).all(), what
    worst = ((got - ref).abs() / tol).max().item() if ref.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance"


def packed_reference(q, k, v, nq, nk, causal, scale, dtype):
    refs, tols, a, b = [], [], 0, 0
    d = q.shape[-1]
    for x, y in zip(nq, nk):
        r = attend(q[a:a + x].double(), k[b:b + y].double(), v[b:b + y].double(), scale, y - x if causal else None)
        refs.append(r[0])
        tols.append(tolerance(*r, d, y, dtype, 2.0 ** -8 if dtype == "bf16" else 2.0 ** -20))
        a, b = a + x, b + y
    return torch.cat(refs), torch.cat(tols)


def run_packed(gpu, nq, nk, heads, kv, d, dtype, causal, scale=None, seed=0, stream=None):
    g = rng(seed)
    behind = 150   # tokens behind the last sequence: no number among the inputs, left as they were in the output
    q = torch.randn(sum(nq) + behind, heads, d, device="cuda", generator=g).to(DT[dtype])
    k = torch.randn(sum(nk) + behind, kv, d, device="cuda", generator=g).to(DT[dtype])
    v = torch.randn(sum(nk) + behind, kv, d, device="cuda", generator=g).to(DT[dtype])
    for x in (q, k, v):
        x[-behind:] = math.nan
    out = torch.full_like(q, 7.0)
    gpu.attention_packed(q, k, v, offsets(nq), offsets(nk), out, causal=causal, scale=scale,
                         stream=torch.cuda.current_stream())
    gpu.synchronize(torch.cuda.current_stream())
    ref, tol = packed_reference(q, k, v, nq, nk, causal, d ** -0.5 if scale is None else scale, dtype)
    assert (out[sum(nq):] == 7.0).all()
    check(out[:sum(nq)], ref, tol, f"{nq} {nk} {heads}/{kv} d{d} {dtype} causal={causal}")


LENGTHS = [
    ([1], [1]),
    ([5, 0, 64, 65, 1], [5, 0, 64, 65, 1]),
    ([127, 128, 129, 31], [127, 128, 129, 31]),
    ([3, 17, 1, 40], [90, 17, 200, 41]),          # more keys than queries
    ([70, 9, 33], [0, 4, 33]),                    # fewer: rows without a key when causal
    ([300], [700]),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk", LENGTHS)
def test_packed_lengths(gpu, nq, nk, causal, dtype):
    run_packed(gpu, nq, nk, 4, 2, 32, dtype, causal, seed=len(nq))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [1, 7, 8, 15, 16, 24, 33, 40, 64, 72, 80, 96, 127, 128])
def test_packed_head_sizes(gpu, d, dtype):
    run_packed(gpu, [37, 100], [50, 100], 2, 1, d, dtype, True, seed=d)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (10, 2), (7, 7), (32, 4), (72, 1), (130, 1)])
def test_packed_groups(gpu, heads, kv, dtype):
    run_packed(gpu, [19, 70], [19, 80], heads, kv, 24, dtype, True, scale=0.3, seed=heads)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_long(gpu, d, causal, dtype):
    run_packed(gpu, [1100, 3, 900], [1100, 1400, 900], 8, 2, d, dtype, causal, seed=d)


@pytest.mark.parametrize("d", [8, 16, 24, 40, 56, 72, 80, 96, 104, 120, 128])
def test_packed_long_head_sizes(gpu, d):
    run_packed(gpu, [300, 555, 128], [300, 600, 128], 4, 2, d, "bf16", True, seed=d)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (10, 2), (7, 7), (40, 1), (128, 1), (129, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_packed_long_groups(gpu, heads, kv, causal):
    run_packed(gpu, [257, 1, 300], [400, 500, 300], heads, kv, 64, "bf16", causal, seed=heads)


@pytest.mark.parametrize("d", [8, 16, 24, 32])
@pytest.mark.parametrize("n", [767, 1700])
def test_packed_small_heads_on_both_sides_of_the_rule(gpu, d, n):
    run_packed(gpu, [n], [n], 2, 1, d, "bf16", True, seed=n + d)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [40, 700])
@pytest.mark.parametrize("d", [16, 64])
@pytest.mark.parametrize("size", [1e5, 1e12, 1e18, 3e19])
def test_packed_scores_beyond_fp32(gpu, n, size, d, dtype):
    """Products near and past FP32's range: rows whose largest score is finite take that key's value (the next
    score is far below), rows whose score overflows are no numbers."""
    q = torch.full((n, 1, d), size, device="cuda").to(DT[dtype])
    k = torch.zeros(n, 1, d, device="cuda").to(DT[dtype])
    k[:, 0, 0] = torch.linspace(0.1, 1, n, device="cuda").to(DT[dtype]) * size
    k[n // 2, 0, 0] = 4 * size
    v = torch.randn(n, 1, d, device="cuda", generator=rng(n)).to(DT[dtype])
    out = torch.empty_like(q)
    gpu.attention_packed(q, k, v, offsets([n]), offsets([n]), out, scale=1.0, stream=torch.cuda.current_stream())
    gpu.synchronize(torch.cuda.current_stream())
    if 4 * size * size * 1.45 < 3e38:
        assert torch.allclose(out.float(), v[n // 2].float().expand(n, 1, d), rtol=2.0 ** -6)
    else:
        assert torch.isnan(out).all()


@pytest.mark.parametrize("d", [1, 15, 16, 31, 32, 33, 64, 72, 127, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_packed_long_fp32(gpu, d, causal):
    run_packed(gpu, [300, 555, 128, 0, 257], [300, 600, 160, 40, 250], 4, 2, d, "f32", causal, seed=d)


@pytest.mark.parametrize("d", [24, 64, 128])
def test_packed_many_long_fp32(gpu, d):   # more blocks than SMs
    run_packed(gpu, [1000, 1201, 900], [1000, 1201, 900], 8, 2, d, "f32", True, seed=d)


@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("powers", [(0, 0, 60), (0, 10, 60), (64, 0, 0), (-64, 0, 30)])
def test_packed_fp32_rows_of_different_powers(gpu, n, causal, powers):
    """Rows of V up to 2^+-60 apart, keys of 2^-10 to 1 of the others, and q and k far from 1 (2^64 among them,
    whose rows are computed from their definition)."""
    shift, below, apart = powers
    g = rng(n + apart)
    q, k, v = (torch.randn(n, h, 48, device="cuda", generator=g) for h in (4, 2, 2))
    q, k = q * 2.0 ** -shift, k * 2.0 ** shift
    k *= torch.exp2(-torch.randint(0, below + 1, (n, 2, 1), device="cuda", generator=g).float())
    v *= torch.exp2(torch.randint(-apart, apart + 1, (n, 2, 1), device="cuda", generator=g).float())
    out = torch.empty_like(q)
    gpu.attention_packed(q, k, v, offsets([n]), offsets([n]), out, causal=causal, stream=torch.cuda.current_stream())
    gpu.synchronize(torch.cuda.current_stream())
    ref, tol = packed_reference(q, k, v, [n], [n], causal, 48 ** -0.5, "f32")
    check(out, ref, tol, f"{n} {powers}")


@pytest.mark.parametrize("n,heads", [(50, 2), (200, 2), (200, 8)])
def test_packed_fp32_later_keys_change_no_bit(gpu, n, heads):
    g = rng(n)
    q, k, v = (torch.randn(n, h, 64, device="cuda", generator=g) for h in (heads, 2, 2))
    outs = []
    for keep in (n, n - 21):
        k[keep:] *= 1e15
        v[keep:] *= 1e30
        outs.append(torch.empty_like(q))
        gpu.attention_packed(q, k, v, offsets([n]), offsets([n]), outs[-1], causal=True,
                             stream=torch.cuda.current_stream())
    gpu.synchronize(torch.cuda.current_stream())
    assert torch.equal(outs[0][:n - 21], outs[1][:n - 21])


@pytest.mark.parametrize("nq,nk", [([1], [256]), ([128, 256], [512, 256]), ([127, 129, 0, 255], [383, 385, 700, 257]),
                                   ([640, 10, 700], [0, 3, 900]), ([2000], [2000]), ([1, 3, 5], [5000, 300, 1025]),
                                   ([1100, 3, 900], [1100, 1400, 900]), ([333] * 40, [333] * 40)])
@pytest.mark.parametrize("causal", [False, True])
def test_packed_long_lengths(gpu, nq, nk, causal):
    for d in (64, 128):
        run_packed(gpu, nq, nk, 4, 2, d, "bf16", causal, seed=d)


def test_packed_growing_scores(gpu):
    """Keys whose scores grow along the sequence: the running maximum moves again and again."""
    n, d = 1500, 64
    for dtype in ("f32", "bf16"):
        g = rng(21)
        q, k, v = (torch.randn(n, 2, d, device="cuda", generator=g) for _ in range(3))
        k = k + q.mean(0, keepdim=True) + torch.arange(n, device="cuda")[:, None, None] / 40 * torch.nn.functional.normalize(q[n // 2:n // 2 + 1], dim=-1)
        q, k, v = (x.to(DT[dtype]) for x in (q, k, v))
        out = torch.empty_like(q)
        s = torch.cuda.current_stream()
        gpu.attention_packed(q, k, v, offsets([n]), offsets([n]), out, stream=s)
        gpu.synchronize(s)
        ref, mag, prod = attend(q.double(), k.double(), v.double(), d ** -0.5)
        check(out, ref, tolerance(ref, mag, prod, d, n, dtype, 2.0 ** -8 if dtype == "bf16" else 2.0 ** -20), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [90, 1000])
def test_packed_strides_and_rows_behind(gpu, dtype, n):
    """Heads before tokens, a fused QKV buffer's strides, and rows past the last sequence left as they were."""
    nq, heads, d = [n, 30], 4, 64
    total = sum(nq) + 5
    g = rng(3)
    qkv = torch.randn(total, 3, heads, d + 8, device="cuda", generator=g).to(DT[dtype])
    q, k, v = (qkv[:, i, :, :d] for i in range(3))
    out = torch.full((heads, total, d), 7.0, device="cuda", dtype=DT[dtype]).transpose(0, 1)
    s = torch.cuda.current_stream()
    gpu.attention_packed(q, k, v, offsets(nq), offsets(nq), out, causal=True, stream=s)
    gpu.synchronize(s)
    ref, tol = packed_reference(q, k, v, nq, nq, True, d ** -0.5, dtype)
    check(out[:sum(nq)], ref, tol)
    assert (out[sum(nq):] == 7.0).all()
    # Every head of K and V the same memory (stride 0).
    k1, v1 = k[:, :1].expand(total, heads, d), v[:, :1].expand(total, heads, d)
    gpu.attention_packed(q, k1, v1, offsets(nq), offsets(nq), out, causal=True, stream=s)
    gpu.synchronize(s)
    ref, tol = packed_reference(q, k1, v1, nq, nq, True, d ** -0.5, dtype)
    check(out[:sum(nq)], ref, tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [100, 1000])
@pytest.mark.parametrize("value", [math.inf, math.nan, -math.inf])
def test_packed_masked_values_never_reach_an_output(gpu, dtype, n, value):
    """Non-finite keys and values behind a row's last key, and in the neighbouring sequences."""
    nq, heads, d = [n, n], 2, 64
    g = rng(4)
    q, k, v = (torch.randn(2 * n, heads, d, device="cuda", generator=g).to(DT[dtype]) for _ in range(3))
    k[n - 3:n] = value                # seen by the last three queries of the first sequence only
    v[n - 2:n, :, ::3] = value
    v[2 * n - 1, 1, 5] = value        # the second sequence's last key: seen by its last query only
    out = torch.empty_like(q)
    s = torch.cuda.current_stream()
    gpu.attention_packed(q, k, v, offsets(nq), offsets(nq), out, causal=True, stream=s)
    gpu.synchronize(s)
    clean = [x.clone() for x in (k, v)]
    for x in clean:
        x[~torch.isfinite(x)] = 0
    ref, tol = packed_reference(q, *clean, nq, nq, True, d ** -0.5, dtype)
    fine = torch.ones(2 * n, dtype=torch.bool, device="cuda")
    fine[n - 3:n] = False
    fine[2 * n - 1] = False
    check(out[fine], ref[fine], tol[fine])
    # A seen infinity or NaN among the values does reach its column, and only that.
    last = out[2 * n - 1, 1].float()
    assert torch.isnan(last[5]) if math.isnan(value) else last[5] == value
    keep = torch.arange(d, device="cuda") != 5
    check(out[2 * n - 1, 1][keep], ref[2 * n - 1, 1][keep], tol[2 * n - 1, 1][keep])
    check(out[2 * n - 1, 0], ref[2 * n - 1, 0], tol[2 * n - 1, 0])


def test_packed_large_scores(gpu):
    """Scores far apart: the softmax is one-hot and nothing overflows."""
    n, d = 200, 64
    for dtype in ("f32", "bf16"):
        g = rng(5)
        q, k, v = (torch.randn(n, 1, d, device="cuda", generator=g).to(DT[dtype]) for _ in range(3))
        q, k = q * 40, k * 40
        out = torch.empty_like(q)
        s = torch.cuda.current_stream()
        gpu.attention_packed(q, k, v, offsets([n]), offsets([n]), out, stream=s)
        gpu.synchronize(s)
        ref, mag, prod = attend(q.double(), k.double(), v.double(), d ** -0.5)
        check(out, ref, tolerance(ref, mag, prod, d, n, dtype, 2.0 ** -8), dtype)


def test_packed_bad_offsets_are_reported_and_stay_in_bounds(gpu):
    g = rng(6)
    q, k, v = (torch.randn(50, 2, 16, device="cuda", generator=g) for _ in range(3))
    s = torch.cuda.current_stream()
    good = offsets([20, 30])
    for bad in ([0, 20, 51], [0, 60, 50], [-4, 20, 50], [0, 30, 20]):
        off = torch.tensor(bad, dtype=torch.int32, device="cuda")
        for a, b in ((off, good), (good, off)):
            gpu.attention_packed(q, k, v, a, b, torch.empty_like(q), causal=True, stream=s)
            with pytest.raises(P.InvalidInput, match="out of range"):
                gpu.synchronize(s)
    gpu.attention_packed(q, k, v, good, good, torch.empty_like(q), stream=s)
    gpu.synchronize(s)   # reported once


def test_packed_wait_expiry_fails_cleanly(gpu):
    """The tcgen05 kernel's waits are bounded: a block whose second step never arrives gives up, and the device
    still computes."""
    with pytest.raises(P.GpuError, match="wait ran out") as info:
        gpu.selftest_wait_expiry(4, 20)
    assert info.value.wait_code != 0
    run_packed(gpu, [600, 700], [600, 700], 4, 2, 128, "bf16", True)


def test_packed_nothing_to_do(gpu):
    s = torch.cuda.current_stream()
    e = torch.empty(0, 2, 16, device="cuda")
    gpu.attention_packed(e, e, e, offsets([]), offsets([]), e, stream=s)
    gpu.attention_packed(e, e, e, offsets([0, 0]), offsets([0, 0]), e, stream=s)
    q = torch.ones(4, 2, 16, device="cuda")
    out = torch.full_like(q, 7.0)
    gpu.attention_packed(q, e, e, offsets([4]), offsets([0]), out, stream=s)   # no keys at all
    gpu.synchronize(s)
    assert (out == 0).all()


# ---------------------------------------------------------------------------
# The cache
# ---------------------------------------------------------------------------

def make_cache(g, lengths, kv, d, page, spare=2, fill=True):
    blocks = [-(-n // page) for n in lengths]
    pages = sum(blocks) + spare
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(1, max(blocks, default=1))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = order[at:at + b]
        at += b
    shape = (pages, kv, page, d)
    k, v = (torch.randint(-128, 128, shape, device="cuda", generator=g).to(torch.int8) for _ in range(2))
    ks, vs = ((0.2 + torch.rand(pages, kv, device="cuda", generator=g) * 3) / 100 for _ in range(2))
    return P.PagedCache(k, v, ks, vs), table


def cache_values(cache, table, i, n, page):
    rows = table[i, : -(-n // page)].long()
    out = []
    for q, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        x = q[rows].double() * s[rows].double()[..., None, None]
        out.append(x.permute(0, 2, 1, 3).reshape(-1, q.shape[1], q.shape[3])[:n])
    return out


def run_cached(gpu, lengths, heads, kv, d, page, dtype, seed=0, scale=None, q=None, cache=None, table=None):
    g = rng(seed)
    if cache is None:
        cache, table = make_cache(g, lengths, kv, d, page)
    if q is None:
        q = torch.randn(len(lengths), heads, d, device="cuda", generator=g).to(DT[dtype])
    out = torch.full_like(q, 7.0)
    s = torch.cuda.current_stream()
    gpu.attention_cached(cache, q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table, out, scale=scale,
                         stream=s)
    gpu.synchronize(s)
    check_cached(out, q, cache, table, lengths, page, dtype, scale)
    return out


def check_cached(out, q, cache, table, lengths, page, dtype, scale=None):
    d = q.shape[-1]
    for i, n in enumerate(lengths):
        k, v = cache_values(cache, table, i, n, page)
        r = attend(q[i:i + 1].double(), k, v, d ** -0.5 if scale is None else scale)
        weight = 2.0 ** -11 if dtype == "bf16" else 2.0 ** -20
        tol = tolerance(*r, d, n, dtype, weight)
        # A weight below FP16's smallest step keeps 2^-31 of the largest one.
        tol = tol + (n * 2.0 ** -31 * v.abs().max() if n else 0)
        check(out[i:i + 1], r[0], tol, f"sequence {i}, length {n}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_cached_lengths(gpu, page, dtype):
    run_cached(gpu, [1, 0, 15, 16, 17, 63, 64, 65, 129, 500, 3000], 4, 2, 64, page, dtype, seed=page)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 56, 64, 72, 80, 104, 112, 120, 128])
def test_cached_head_sizes(gpu, d, dtype):
    run_cached(gpu, [33, 200], 6, 2, d, 16, dtype, seed=d)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 1), (8, 1), (9, 1), (17, 1), (32, 2), (21, 3)])
def test_cached_groups(gpu, heads, kv, dtype):
    run_cached(gpu, [70, 1, 0, 333], heads, kv, 48, 32, dtype, seed=heads, scale=0.2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [2047, 5000, 20001])
def test_cached_few_long_sequences(gpu, n, dtype):
    """One and two sequences: the range is split over a cluster."""
    run_cached(gpu, [n], 4, 1, 128, 64, dtype, seed=n)
    run_cached(gpu, [n, 3], 8, 2, 64, 16, dtype, seed=n + 1)


def test_cached_many_sequences(gpu):
    r = np.random.default_rng(0)
    run_cached(gpu, [int(x) for x in r.integers(0, 90, 300)], 4, 2, 32, 16, "bf16")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_cached_scales_far_apart(gpu, dtype):
    """Pages of zeros, of tiny and of large values next to each other; queries from 1e-6 to 1e4."""
    g = rng(9)
    lengths, page, d = [160, 100, 64], 16, 64
    cache, table = make_cache(g, lengths, 2, d, page)
    at = torch.arange(cache.k.shape[0], device="cuda")
    cache.v_scales.copy_((10.0 ** (-(at % 4).float()))[:, None] * cache.v_scales)
    cache.v_scales[table[0, 0].long()] = 0
    cache.k_scales[table[1, 1].long()] = 0
    q = torch.randn(3, 4, d, device="cuda", generator=g)
    q[1] *= 1e-6
    q[2] *= 30
    q[0, 0] = 0
    run_cached(gpu, lengths, 4, 2, d, page, dtype, q=q.to(DT[dtype]), cache=cache, table=table)


def test_cached_strides(gpu):
    g = rng(10)
    lengths, page, d, heads = [40, 100], 32, 64, 6
    cache, table = make_cache(g, lengths, 2, d, page)
    wide = torch.full((2, 9), 10 ** 6, dtype=torch.int32, device="cuda")   # entries past the lengths are not read
    wide[:, :table.shape[1]] = table
    q = torch.randn(heads, 2, d + 3, device="cuda", generator=g).bfloat16().transpose(0, 1)[..., 1:d + 1]
    out = torch.full((2, heads + 1, d + 5), 7.0, device="cuda").bfloat16()
    s = torch.cuda.current_stream()
    gpu.attention_cached(cache, q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), wide, out[:, :heads, 3:d + 3],
                         stream=s)
    gpu.synchronize(s)
    check_cached(out[:, :heads, 3:d + 3], q, cache, table, lengths, page, "bf16")
    assert (out[:, heads] == 7).all() and (out[..., :3] == 7).all() and (out[..., d + 3:] == 7).all()


def test_cached_bad_tables_and_lengths_are_reported(gpu):
    g = rng(11)
    cache, table = make_cache(g, [40, 100], 2, 64, 16)
    q = torch.randn(2, 4, 64, device="cuda", generator=g)
    s = torch.cuda.current_stream()
    for lengths, entry in (([40, 1000], None), ([-1, 100], None), ([40, 100], -1), ([40, 100], cache.k.shape[0]),
                           ([40, 100], 2 ** 31 - 1), ([40, 100], -2 ** 31)):
        t = table.clone()
        if entry is not None:
            t[1, 3] = entry
        else:   # a length past the table reads its last entries: keep those good
            t[t < 0] = 0
        gpu.attention_cached(cache, q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), t, torch.empty_like(q), stream=s)
        with pytest.raises(P.InvalidInput, match="out of range"):
            gpu.synchronize(s)
    gpu.synchronize(s)


def append_reference(cache, table, x, y, n, held, page):
    """Float64 append, in place on clones; returns the cache that should be."""
    out = []
    for q, s, new in ((cache.k, cache.k_scales, x), (cache.v, cache.v_scales, y)):
        q, s = q.cpu().numpy().copy(), s.cpu().numpy().copy()
        new, t, at = new.float().cpu().numpy(), table.cpu().numpy(), 0
        for i, (a, h) in enumerate(zip(n, held)):
            pos = h
            while pos < h + a:
                b, lo = t[i, pos // page], pos % page
                hi = min(page, lo + h + a - pos)
                part = new[at:at + hi - lo]                                  # [tokens, heads, d]
                before = s[b].copy() if lo else np.zeros_like(s[b])
                now = np.maximum(before, np.abs(part).max((0, 2)) * np.float32(1 / 127))
                grown = (now > before)[:, None, None]
                with np.errstate(all="ignore"):
                    again = np.rint(q[b, :, :lo].astype(np.float64) * before.astype(np.float64)[:, None, None]
                                    / now.astype(np.float64)[:, None, None])
                    fresh = np.rint(part.transpose(1, 0, 2).astype(np.float64) / now.astype(np.float64)[:, None, None])
                again = np.where(grown, again, q[b, :, :lo])
                fresh = np.where((now > 0)[:, None, None], fresh, 0).clip(-127, 127)
                q[b, :, :lo], q[b, :, lo:hi], s[b] = again, fresh, now
                pos, at = pos + hi - lo, at + hi - lo
        out += [q, s]
    return out


def run_append(gpu, n, held, kv, d, page, dtype, seed=0, new=None, cache=None, table=None):
    g = rng(seed)
    if cache is None:
        cache, table = make_cache(g, [a + h for a, h in zip(n, held)], kv, d, page)
        for q in (cache.k, cache.v):
            q.clamp_(min=-127)
    if new is None:
        new = [torch.randn(sum(n), kv, d, device="cuda", generator=g).to(DT[dtype]) * 1.5 for _ in range(2)]
    want = append_reference(cache, table, *new, n, held, page)
    s = torch.cuda.current_stream()
    gpu.cache_append(cache, *new, offsets(n), torch.tensor(held, dtype=torch.int32, device="cuda"), table, stream=s)
    gpu.synchronize(s)
    for got, ref, name in zip((cache.k, cache.k_scales, cache.v, cache.v_scales), want, ("k", "k scales", "v", "v scales")):
        np.testing.assert_array_equal(got.cpu().numpy(), ref, err_msg=name)
    return cache, table


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page,d,kv", [(16, 64, 2), (32, 24, 3), (64, 128, 1), (128, 128, 2), (16, 8, 1)])
def test_append_is_exact(gpu, page, d, kv, dtype):
    """Integers and scales equal the definition's: new, part-filled and several pages, lengths 0 and 1."""
    run_append(gpu, [1, 0, 5, page, page + 1, 3 * page + 7, 1, 200], [0, 3, page - 1, 0, 7, page, 2 * page - 1, 15], kv, d, page,
               dtype, seed=page + d)


def test_append_rounds_ties_to_even(gpu):
    """A scale that is a power of two puts every half on a tie."""
    page, d = 16, 64
    x = torch.arange(16 * d, device="cuda", dtype=torch.float32).view(16, 1, d) % 254 - 127
    x = x + 0.5 * (x < 127) * (x > -127)
    x = x.clamp(-127, 127)
    x[0, 0, 0] = 127                        # scale 127 / 127
    for unit in (1.0, 2.0 ** -20, 2.0 ** 30):
        cache, _ = run_append(gpu, [16], [0], 1, d, page, "f32", new=[x * unit, x * unit])
    # The same step as a part-filled page's: integers 2 n + 1 halve to ties when the scale doubles.
    g = rng(1)
    cache, table = make_cache(g, [page], 1, d, page)
    cache.k.clamp_(min=-127)
    cache.v.clamp_(min=-127)
    cache.k_scales.fill_(1.0)
    cache.v_scales.fill_(1.0)
    new = torch.full((1, 1, d), 254.0, device="cuda")
    run_append(gpu, [1], [15], 1, d, page, "f32", new=[new, -new], cache=cache, table=table)


def test_append_near_ties(gpu):
    """Quotients one step of FP32 to either side of a half, and far below it."""
    page, d = 16, 64
    r = np.random.default_rng(2)
    scale = np.float32(r.uniform(0.01, 3))
    half = (r.integers(-126, 126, 15 * d) + 0.5).astype(np.float64) * float(scale * np.float32(1 / 127) * 1)
    x = half.astype(np.float32)
    x[::3] = np.nextafter(x[::3], np.float32(9))
    x[1::3] = np.nextafter(x[1::3], np.float32(-9))
    x = np.concatenate([np.full(d, scale, np.float32), x]).reshape(16, 1, d)
    t = torch.from_numpy(x).cuda()
    run_append(gpu, [16], [0], 1, d, page, "f32", new=[t, -t])
    z = torch.zeros_like(t)
    run_append(gpu, [16], [0], 1, d, page, "f32", new=[z, t * 1e-38])


def test_append_strided_sources_and_other_pages_untouched(gpu):
    g = rng(12)
    n, held, kv, d, page = [20, 3], [5, 16], 2, 40, 16
    src = torch.randn(kv, 23, 2 * d + 1, device="cuda", generator=g)
    k, v = src[..., :d].transpose(0, 1), src[..., d + 1:].transpose(0, 1)
    cache, table = make_cache(g, [25, 19], kv, d, page, spare=4)
    cache.k.clamp_(min=-127)
    cache.v.clamp_(min=-127)
    run_append(gpu, n, held, kv, d, page, "f32", new=[k, v], cache=cache, table=table)


def test_append_marks_pages_that_are_not_finite(gpu):
    page, d = 16, 16
    g = rng(13)
    for value in (math.nan, math.inf, -math.inf):
        cache, table = make_cache(g, [20], 2, d, page)
        x = torch.randn(20, 2, d, device="cuda", generator=g)
        x[17, 1, 3] = value
        s = torch.cuda.current_stream()
        zero = torch.zeros(1, dtype=torch.int32, device="cuda")
        gpu.cache_append(cache, x, x, offsets([20]), zero, table, stream=s)
        k, v = torch.empty_like(x), torch.empty_like(x)
        gpu.cache_read(cache, k, v, offsets([20]), zero, table, stream=s)
        gpu.synchronize(s)
        assert not torch.isfinite(cache.k_scales[table[0, 1].long(), 1])
        assert torch.isnan(k[16:, 1]).all() and torch.isfinite(k[:16]).all() and torch.isfinite(k[:, 0]).all()
        # A new first token starts the page afresh.
        gpu.cache_append(cache, x[:1], x[:1], offsets([1]), zero + 16, table, stream=s)
        gpu.synchronize(s)
        assert torch.isfinite(cache.k_scales[table[0, 1].long()]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page,d", [(16, 64), (64, 24), (128, 128)])
def test_read(gpu, page, d, dtype):
    g = rng(14)
    lengths, first, n = [100, 7, 300, 0, 1], [30, 0, 290, 0, 0], [70, 7, 10, 0, 1]
    cache, table = make_cache(g, lengths, 2, d, page)
    total = sum(n)
    k = torch.full((total + 2, 2, d), 7.0, device="cuda", dtype=DT[dtype])
    v = torch.full((2, total + 2, d), 7.0, device="cuda", dtype=DT[dtype]).transpose(0, 1)
    s = torch.cuda.current_stream()
    gpu.cache_read(cache, k, v, offsets(n), torch.tensor(first, dtype=torch.int32, device="cuda"), table, stream=s)
    gpu.synchronize(s)
    at = 0
    for i, (f, x) in enumerate(zip(first, n)):
        want = cache_values(cache, table, i, f + x, page)
        for got, ref in zip((k, v), want):   # one product, rounded to FP32 and then to the type
            check(got[at:at + x], ref[f:], ref[f:].abs() * (2.0 ** -24 + HALF_STEP[dtype] * (1 + 2.0 ** -20)) + 1e-40)
        at += x
    assert (k[total:] == 7).all() and (v[total:] == 7).all()


def test_append_and_read_report_bad_arguments(gpu):
    g = rng(15)
    cache, table = make_cache(g, [40, 30], 2, 16, 16)
    keep = [x.clone() for x in (cache.k, cache.v, cache.k_scales, cache.v_scales)]
    x = torch.randn(10, 2, 16, device="cuda", generator=g)
    s = torch.cuda.current_stream()
    i32 = dict(dtype=torch.int32, device="cuda")
    bad_table = torch.full_like(table, cache.k.shape[0])
    for off, pos, t in (([0, 5, 10], [-1, -9], table), ([0, 5, 10], [1000, 47], table), ([0, 5, 10], [0, 0], bad_table),
                        ([0, 5, 10], [0, 0], -bad_table), ([0, 5, 10], [2 ** 31 - 1, 2 ** 31 - 3], table)):
        gpu.cache_append(cache, x, x, torch.tensor(off, **i32), torch.tensor(pos, **i32), t, stream=s)
        with pytest.raises(P.InvalidInput, match="out of range"):
            gpu.synchronize(s)
        out = torch.full_like(x, 7.0)
        gpu.cache_read(cache, out, out.clone(), torch.tensor(off, **i32), torch.tensor(pos, **i32), t, stream=s)
        with pytest.raises(P.InvalidInput, match="out of range"):
            gpu.synchronize(s)
        assert (out == 7).all()
    for got, was in zip((cache.k, cache.v, cache.k_scales, cache.v_scales), keep):
        assert torch.equal(got, was)


# ---------------------------------------------------------------------------
# Logit rules
# ---------------------------------------------------------------------------

def rules_reference(x, history, n, rep, pres, freq, bias, mask, index):
    y = x.double().clone()
    mag = y.abs()
    edge = np.concatenate([[0], np.cumsum(n)]) if history is not None else None
    for r in range(x.shape[0]):
        if history is not None:
            ids, times = torch.unique(history[edge[r]:edge[r + 1]].long(), return_counts=True)
            z = y[r, ids]
            if rep is not None:
                z = torch.where(z > 0, z / rep[r].double(), z * rep[r].double())
            m = z.abs().maximum(mag[r, ids])
            for p, t in ((freq, times), (pres, 1)):
                if p is not None:
                    z = z - p[r].double() * t
                    m = m + (p[r].double() * t).abs()
            y[r, ids], mag[r, ids] = z, m
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    if mask is not None:
        bits = ((mask[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).flatten(1)[:, :x.shape[1]] == 0
        for r in range(x.shape[0]):
            state = 0 if index is None else int(index[r])
            if state >= 0:
                y[r, bits[state]] = -math.inf
    return y, mag


def run_rules(gpu, rows, vocab, dtype, history=0, penalties=True, bias=True, states=0, index=True, pad=0, shift=0, inplace=False,
              seed=0):
    g = rng(seed)
    r = np.random.default_rng(seed)
    base = torch.randn(rows, vocab + pad + shift, device="cuda", generator=g).to(DT[dtype]) * 3
    x = base[:, shift:shift + vocab]
    whole = base.clone()
    kw, n, ids = {}, None, None
    if history:
        n = [int(v) for v in r.integers(0, history + 1, rows)]
        n[0] = 0
        ids = torch.from_numpy(r.integers(0, max(1, min(vocab, history // 2)), sum(n)).astype(np.int32)).cuda()
        kw = dict(history=ids, history_offsets=offsets(n))
        if penalties:
            kw.update(repetition=1 + torch.rand(rows, device="cuda", generator=g), presence=torch.rand(rows, device="cuda", generator=g),
                      frequency=torch.rand(rows, device="cuda", generator=g) - 0.5)
    if bias:
        kw["bias"] = torch.randn(vocab, device="cuda", generator=g)
    if states:
        kw["mask"] = torch.randint(-2 ** 31, 2 ** 31, (states, -(-vocab // 32) + 1), device="cuda", generator=g).to(torch.int32)
        kw["mask"][0] = 0            # a state that allows nothing
        if index:
            kw["mask_index"] = torch.randint(-1, states, (rows,), device="cuda", generator=g, dtype=torch.int32)
    want, mag = rules_reference(x, ids, n, kw.get("repetition"), kw.get("presence"), kw.get("frequency"), kw.get("bias"),
                                kw.get("mask"), kw.get("mask_index"))
    out = x if inplace else torch.empty(rows, vocab, device="cuda", dtype=DT[dtype])
    s = torch.cuda.current_stream()
    assert gpu.logit_rules(x, out, stream=s, **kw) is out
    gpu.synchronize(s)
    gone = torch.isinf(want)
    assert torch.equal(torch.isinf(out) & (out < 0), gone)
    # Four FP32 roundings of terms no larger than `mag`, then the type's.
    tol = mag * 2.0 ** -22 + HALF_STEP[dtype] * (want.abs() + mag * 2.0 ** -22) + 1e-30
    check(out[~gone], want[~gone], tol[~gone], f"{rows} x {vocab} {dtype}")
    if inplace and pad:
        assert torch.equal(base[:, shift + vocab:], whole[:, shift + vocab:])
        assert torch.equal(base[:, :shift], whole[:, :shift])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [1, 31, 33, 100, 6906, 6907, 18710, 40001])
def test_rules_vocabularies(gpu, vocab, dtype):
    run_rules(gpu, 5, vocab, dtype, states=3, seed=vocab)
    run_rules(gpu, 5, vocab, dtype, history=300, states=3, seed=vocab + 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 7, 300])
def test_rules_rows(gpu, rows, dtype):
    run_rules(gpu, rows, 1000, dtype, states=1, index=False, seed=rows)
    run_rules(gpu, rows, 1000, dtype, history=50, states=4, seed=rows)
    run_rules(gpu, rows, 1000, dtype, history=50, penalties=False, bias=False, seed=rows)
    run_rules(gpu, rows, 1000, dtype, bias=False, seed=rows)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 0), (2, 2), (4, 4), (3, 5), (8, 8)])
def test_rules_strides_in_place(gpu, pad, shift, dtype):
    """Every alignment of rows; columns outside the logits survive."""
    run_rules(gpu, 6, 2050, dtype, history=100, states=2, pad=pad, shift=shift, inplace=True, seed=pad)
    run_rules(gpu, 6, 2050, dtype, states=2, pad=pad, shift=shift, inplace=True, seed=pad)


def test_rules_long_history_and_many_rows(gpu):
    run_rules(gpu, 3, 50, "f32", history=20000, seed=1)
    run_rules(gpu, 66000, 8, "f32", history=2, seed=2)


def test_rules_non_finite_logits(gpu):
    """A masked NaN or infinity becomes -infinity; an allowed one stays."""
    x = torch.tensor([[math.nan, math.inf, -math.inf, 1.0]] * 2, device="cuda")
    mask = torch.tensor([[0b1100]], dtype=torch.int32, device="cuda")
    s = torch.cuda.current_stream()
    out = gpu.logit_rules(x, torch.empty_like(x), mask=mask, stream=s)
    gpu.synchronize(s)
    assert torch.equal(out, torch.tensor([[-math.inf, -math.inf, -math.inf, 1.0]] * 2, device="cuda"))
    out = gpu.logit_rules(x, torch.empty_like(x), bias=torch.ones(4, device="cuda"), stream=s)
    gpu.synchronize(s)
    assert torch.isnan(out[:, 0]).all() and (out[:, 1] == math.inf).all() and (out[:, 2] == -math.inf).all()


def test_rules_report_bad_ids_states_and_offsets(gpu):
    i32 = dict(dtype=torch.int32, device="cuda")
    x = torch.randn(2, 100, device="cuda")
    s = torch.cuda.current_stream()
    off = torch.tensor([0, 2, 4], **i32)
    ones = torch.ones(2, device="cuda")
    mask = torch.full((2, 4), -1, **i32)
    for kw in (dict(history=torch.tensor([1, 100, 5, 5], **i32), history_offsets=off, presence=ones),
               dict(history=torch.tensor([1, -1, 5, 5], **i32), history_offsets=off, presence=ones),
               dict(history=torch.tensor([1, 2, 5, 5], **i32), history_offsets=off + 1, presence=ones),
               dict(mask=mask, mask_index=torch.tensor([0, 2], **i32)),
               dict(mask=mask, mask_index=torch.tensor([-2, 0], **i32))):
        gpu.logit_rules(x, torch.empty_like(x), stream=s, **kw)
        with pytest.raises(P.InvalidInput, match="out of range"):
            gpu.synchronize(s)


# ---------------------------------------------------------------------------
# Streams, graphs, and a run of the operators together
# ---------------------------------------------------------------------------

def test_default_stream_is_the_handles_own(gpu):
    q = torch.randn(40, 2, 16, device="cuda")
    off = offsets([40])
    torch.cuda.synchronize()
    out = torch.full_like(q, 7.0)
    torch.cuda.synchronize()
    gpu.attention_packed(q, q, q, off, off, out)
    gpu.synchronize()
    ref, tol = packed_reference(q, q, q, [40], [40], False, 0.25, "f32")
    check(out, ref, tol)


def test_two_streams_at_once(gpu):
    """Calls on two streams do not share anything."""
    g = rng(20)
    lengths = [4000, 900]
    cache, table = make_cache(g, lengths, 2, 64, 16)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    qs = [torch.randn(2, 8, 64, device="cuda", generator=g) for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(20)] for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(20):
        for q, o, s in zip(qs, outs, streams):
            gpu.attention_cached(cache, q, n, table, o[i], stream=s)
    for s in streams:
        gpu.synchronize(s)
    for q, o in zip(qs, outs):
        check_cached(o[0], q, cache, table, lengths, 16, "f32")
        assert all(torch.equal(o[0], x) for x in o[1:])   # and repeat bit for bit


class Decoder:
    """Prompts through the packed attention, their keys and values into the cache, then one token a step: the
    cached attention, logits against a table of vectors, the logit rules and the arg-max."""

    def __init__(self, gpu, dtype, seed):
        g = rng(seed)
        self.gpu, self.dtype, self.page, self.d, self.heads, self.kv, self.vocab = gpu, dtype, 16, 64, 4, 2, 500
        t = DT[dtype]
        self.prompts = [33, 1, 70, 16]
        total = sum(self.prompts)
        self.q = torch.randn(total, self.heads, self.d, device="cuda", generator=g).to(t)
        self.k = torch.randn(total, self.kv, self.d, device="cuda", generator=g).to(t)
        self.v = torch.randn(total, self.kv, self.d, device="cuda", generator=g).to(t)
        self.steps = 20
        self.cache, self.table = make_cache(g, [n + self.steps for n in self.prompts], self.kv, self.d, self.page)
        b = len(self.prompts)
        self.words = torch.randn(self.vocab, self.heads * self.d, device="cuda", generator=g) * 0.2
        self.new = torch.randn(self.vocab, 2, self.kv, self.d, device="cuda", generator=g).to(t)
        self.ask = torch.randn(self.vocab, self.heads, self.d, device="cuda", generator=g).to(t)
        self.lengths = torch.tensor(self.prompts, dtype=torch.int32, device="cuda")
        self.one = offsets([1] * b)
        self.token = torch.arange(b, device="cuda")
        self.out = torch.empty(b, self.heads, self.d, device="cuda", dtype=t)
        self.logits = torch.empty(b, self.vocab, device="cuda")
        # Each row's history: room for every step, the unwritten ones padded with its own first id.
        self.history = torch.zeros(b, self.steps, dtype=torch.int32, device="cuda")
        self.history_offsets = offsets([self.steps] * b)
        self.presence = torch.full((b,), 5.0, device="cuda")
        self.mask = torch.full((1, 16), -1, dtype=torch.int32, device="cuda")
        self.mask[0, :8] = 0x55555555

    def prompt(self):
        off, out, s = offsets(self.prompts), torch.empty_like(self.q), torch.cuda.current_stream()
        self.gpu.attention_packed(self.q, self.k, self.v, off, off, out, causal=True, stream=s)
        self.gpu.cache_append(self.cache, self.k, self.v, off, torch.zeros_like(self.lengths), self.table, stream=s)
        return out

    def step(self, i=None):
        """One token; in a captured step the position in the history is `self.at`."""
        s = torch.cuda.current_stream()
        kv = self.new[self.token]
        self.gpu.cache_append(self.cache, kv[:, 0], kv[:, 1], self.one, self.lengths, self.table, stream=s)
        self.lengths += 1
        self.gpu.attention_cached(self.cache, self.ask[self.token], self.lengths, self.table, self.out, stream=s)
        torch.matmul(self.out.float().flatten(1), self.words.T, out=self.logits)
        self.gpu.logit_rules(self.logits, self.logits, history=self.history.view(-1), history_offsets=self.history_offsets,
                             presence=self.presence, mask=self.mask, stream=s)
        self.token.copy_(self.logits.argmax(-1))
        self.history.copy_(torch.cat([self.history[:, 1:], self.token[:, None].int()], 1))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompt_then_steps(gpu, dtype):
    x = Decoder(gpu, dtype, 30)
    out = x.prompt()
    gpu.synchronize(torch.cuda.current_stream())
    ref, tol = packed_reference(x.q, x.k, x.v, x.prompts, x.prompts, True, x.d ** -0.5, dtype)
    check(out, ref, tol)
    for i in range(x.steps):
        before, history = x.token.clone(), x.history.clone()
        x.step()
        gpu.synchronize(torch.cuda.current_stream())
        lengths = [n + i + 1 for n in x.prompts]
        check_cached(x.out, x.ask[before], x.cache, x.table, lengths, x.page, dtype)
        # The cache holds the newest values to half of its scale's step.
        for b, n in enumerate(lengths):
            at = x.table[b, (n - 1) // x.page].long()
            got = x.cache.k[at, :, (n - 1) % x.page].float() * x.cache.k_scales[at][:, None]
            assert ((got - x.new[before[b], 0].float()).abs() <= 0.5001 * x.cache.k_scales[at][:, None]).all()
        want, mag = rules_reference(x.out.float().flatten(1) @ x.words.T, history.view(-1), [x.steps] * 4, None, x.presence, None,
                                    None, x.mask, None)
        assert torch.equal(want.argmax(-1), x.token) or (want.amax(-1) - want.gather(1, x.token[:, None])[:, 0]).max() < 1e-4
        assert (x.token < 256).logical_and(x.token % 2 == 1).sum() == 0   # only what the mask allows
    # The prompt's prefix read back from the cache answers as the cache does.
    n = [5, 1, 70, 16]
    k = torch.empty(sum(n), x.kv, x.d, device="cuda", dtype=DT[dtype])
    v = torch.empty_like(k)
    s = torch.cuda.current_stream()
    gpu.cache_read(x.cache, k, v, offsets(n), torch.zeros(4, dtype=torch.int32, device="cuda"), x.table, stream=s)
    q = x.ask[:4]
    a = gpu.attention_packed(q, k, v, x.one, offsets(n), torch.empty_like(q), causal=True, stream=s)
    b = gpu.attention_cached(x.cache, q, torch.tensor(n, dtype=torch.int32, device="cuda"), x.table, torch.empty_like(q), stream=s)
    gpu.synchronize(s)
    # Reading back rounds the values to the type once more: at most 2^-8 (2^-24) of each key and value.
    assert (a.float() - b.float()).abs().max() <= (0.08 if dtype == "bf16" else 1e-4)


def test_captured_steps_equal_eager_ones(gpu):
    eager, graphed = Decoder(gpu, "bf16", 31), Decoder(gpu, "bf16", 31)
    for x in (eager, graphed):
        x.prompt()
        x.step()   # warm-up: the library's handles of torch are made outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.step()
    for _ in range(8):
        eager.step()
        graph.replay()
    gpu.synchronize(torch.cuda.current_stream())
    assert torch.equal(eager.history, graphed.history) and torch.equal(eager.out, graphed.out)
    assert torch.equal(eager.lengths, graphed.lengths)
    assert torch.equal(eager.cache.k, graphed.cache.k) and torch.equal(eager.cache.v_scales, graphed.cache.v_scales)


# ---------------------------------------------------------------------------
# The recognizer's use of them
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("size", ["tiny", "small"])
def test_recognizer_class_rules(gpu, weights_file, size):
    from ppocr_b200 import seeded

    rec = P.Recognizer.load(gpu, weights_file("rec", size, "conditioned"), size, (3, 3, 48, 96))
    x = seeded.rec_batch(3, 96, seed=5)
    plain = rec.forward_ctc(x)
    logits = rec.forward_logits(x).astype(np.float64)
    classes = logits.shape[-1]
    r = np.random.default_rng(7)
    bias = r.normal(0, 1, classes).astype(np.float32)
    allowed = r.random(classes) < 0.3
    allowed[0] = True
    one = np.zeros(classes, bool)
    one[17] = True
    for b, a in ((bias, None), (None, allowed), (bias, allowed), (None, one)):
        idx, prob, margin = rec.forward_ctc(x, bias=b, allowed=a)
        z = logits + (0 if b is None else b)
        if a is not None:
            z = np.where(a, z, -np.inf)
        e = np.exp(z - z.max(-1, keepdims=True))
        p = e / e.sum(-1, keepdims=True)
        assert (p.max(-1) - np.take_along_axis(p, idx[..., None], -1)[..., 0] <= 1e-6).all()
        assert a is None or a[idx].all()
        np.testing.assert_allclose(prob, p.max(-1), atol=2e-6)
        if a is one:
            assert (idx == 17).all() and (margin == np.finfo(np.float32).max).all()
        else:
            top = np.sort(z, -1)
            np.testing.assert_allclose(margin, top[..., -1] - top[..., -2], atol=1e-4)
    for was, now in zip(plain, rec.forward_ctc(x)):
        np.testing.assert_array_equal(was, now)   # a later plain call is not held to the rules
    with pytest.raises(P.InvalidInput, match="no class"):
        rec.forward_ctc(x, allowed=np.zeros(classes, bool))
    with pytest.raises(P.InvalidInput, match="finite"):
        rec.forward_ctc(x, bias=np.full(classes, np.nan, np.float32))
    with pytest.raises(P.InvalidInput, match="shape"):
        rec.forward_ctc(x, allowed=np.ones(classes - 1, bool))


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
@pytest.mark.parametrize("size,width", [("small", 12160), ("medium", 8000)])
def test_recognizer_of_very_wide_lines(gpu, weights_file, size, width, precision):
    """Lines whose K and V do not fit in shared memory: the encoder's attention is the packed one."""
    from ppocr_b200 import seeded

    rec = P.Recognizer.load(gpu, weights_file("rec", size, "conditioned"), size, (1, 3, 48, width), precision=precision,
                            keep_tensors=True)
    out = rec.forward(seeded.rec_batch(1, width, seed=6))
    assert np.isfinite(out.values).all()
    block = "head.encoder.svtr_block.0"
    names = {t["name"]: t["shape"] for t in rec.tensors()}
    qkv = torch.from_numpy(rec.read_tensor(block + ".qkv")).double()
    got = torch.from_numpy(rec.read_tensor(block + ".attn")).double()
    t, hidden = names[block + ".attn"][2], names[block + ".attn"][3]
    d = hidden // 8
    qkv, got = qkv.reshape(t, 3, 8, d), got.reshape(t, 8, d)
    dtype = "bf16" if precision == "bf16" else "f32"
    r = attend(qkv[:, 0], qkv[:, 1], qkv[:, 2], d ** -0.5)
    check(got, r[0], tolerance(*r, d, t, dtype, 2.0 ** -8 if dtype == "bf16" else 2.0 ** -20), size)
