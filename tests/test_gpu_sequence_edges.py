"""Sequence operators at the ends of their ranges, against plain float64 implementations.

Tolerances are those of the sequence operators' other tests, the sums of the roundings that the kernels document;
what a test adds to them stands beside it.
"""

import math

import pytest

import ppocr_b200 as P

torch = pytest.importorskip("torch")
import test_gpu_sequence_ops as ops  # noqa: E402

pytestmark = pytest.mark.gpu

DT, HALF_STEP = ops.DT, ops.HALF_STEP


def packed(gpu, q, k, v, nq, nk, causal=False, scale=None):
    s = torch.cuda.current_stream()
    out = torch.full_like(q, 7.0)
    gpu.attention_packed(q, k, v, ops.offsets(nq), ops.offsets(nk), out, causal=causal, scale=scale, stream=s)
    gpu.synchronize(s)
    return out


# ---------------------------------------------------------------------------
# Packed attention: masked keys and values, whatever they hold
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("n", [100, 1000])
@pytest.mark.parametrize("causal", [False, True])
def test_packed_masked_finite_values_change_no_bit(gpu, n, d, causal, dtype):
    """Large finite values behind a row's last key, and keys and values in the sequence between and behind the last
    one."""
    g = ops.rng(n + d)
    lengths, behind = [n, n - 3, n], 150
    q, k, v = (torch.randn(sum(lengths) + behind, h, d, device="cuda", generator=g).to(DT[dtype]) for h in (4, 2, 2))
    masked = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    masked[n:2 * n - 3] = True                     # all of the middle sequence
    masked[sum(lengths):] = True
    others, rows = masked.clone(), ~masked
    if causal:                                     # the last values of the first sequence: seen by its last queries
        masked[n - 3:n] = True
        rows[n - 3:n] = False
    huge = torch.where(torch.rand(v.shape, device="cuda", generator=g) < 0.5, 3e38, -3e38).to(DT[dtype])
    outs = []
    for fill in (torch.zeros_like(huge), huge):
        kk, vv = k.clone(), v.clone()
        kk[others], vv[masked] = fill[others], fill[masked]
        outs.append(packed(gpu, q, kk, vv, lengths, lengths, causal))
    assert torch.isfinite(outs[0][rows]).all()
    assert torch.equal(outs[0][rows], outs[1][rows])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [40, 1000])
@pytest.mark.parametrize("below", [160, 300, 100000])
def test_packed_keys_far_below_weigh_nothing(gpu, n, below, dtype):
    """Visible keys whose scores lie `below` powers of two under the others' have no weight, however large their
    values (2^-160 of 1e38 is 1e-10)."""
    d = 64
    g = ops.rng(n)
    q, k, v = (torch.randn(n, 2, d, device="cuda", generator=g) for _ in range(3))
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    far = torch.rand(n, device="cuda", generator=g) < 0.5
    far[n // 3] = False
    k[far, :, 0] = -float(below) * 8 * math.log(2) * 1.1   # scale 1 / 8; the other products stay within a tenth
    v[far] = 1e38
    q, k, v = (x.to(DT[dtype]) for x in (q, k, v))
    out = packed(gpu, q, k, v, [n], [n])
    ref, mag, prod = ops.attend(q.double(), k[~far].double(), v[~far].double(), d ** -0.5)
    ops.check(out, ref, ops.tolerance(ref, mag, prod, d, n, dtype, 2.0 ** -8 if dtype == "bf16" else 2.0 ** -20) + 1e-9)


# ---------------------------------------------------------------------------
# Bad offsets
# ---------------------------------------------------------------------------

def read_by_hand(cache, table, offsets, first, total, page, kv, d):
    """What a read may write: each token by the sequence whose clamped offsets hold it, None elsewhere."""
    k = [None] * total
    for i in range(len(offsets) - 1):
        a = min(max(offsets[i], 0), total)
        b = min(max(offsets[i + 1], a), total)
        for t in range(a, b):
            pos = first[i] + t - a
            k[t] = cache.k[table[i, pos // page].long(), :, pos % page].float() * cache.k_scales[table[i, pos // page].long()][:, None]
    return k


@pytest.mark.parametrize("bad", [[-4, 10, 20], [0, 10, 25], [-2 ** 31, 10, 20], [0, 2 ** 31 - 1, 20], [-2 ** 31, 2 ** 31 - 1, 20],
                                 [0, 10, -2 ** 31], [5, 3, 20]])
def test_read_clamps_and_reports_bad_offsets(gpu, bad):
    """A token of the output is what the clamped offsets say, or left as it was; the next synchronize reports them."""
    g = ops.rng(3)
    page, kv, d, total = 16, 2, 16, 20
    cache, table = ops.make_cache(g, [60, 60], kv, d, page)
    first = [3, 7]
    s = torch.cuda.current_stream()
    i32 = dict(dtype=torch.int32, device="cuda")
    k, v = (torch.full((total, kv, d), 7.0, device="cuda") for _ in range(2))
    gpu.cache_read(cache, k, v, torch.tensor(bad, **i32), torch.tensor(first, **i32), table, stream=s)
    with pytest.raises(P.InvalidInput, match="out of range"):
        gpu.synchronize(s)
    want = read_by_hand(cache, table, bad, first, total, page, kv, d)
    for t in range(total):
        same = want[t] is not None and torch.equal(k[t], want[t])
        assert same or ((k[t] == 7).all() and (v[t] == 7).all()), t


BAD_OFFSETS = [[0, 3000, 100, 4000], [0, 100, 50, 120], [0, 4000, 3999, 4000, 4000], [0, 10, 4001, 20, 4000],
               [0, 10, -1, 20, 4000], [4000, 4000, 2 ** 31 - 1], [0, 4000, 4000, -2 ** 31, 4000, 4000]]


@pytest.mark.parametrize("bad", BAD_OFFSETS)
def test_every_bad_offset_is_reported(gpu, bad):
    """Also those of sequences that no block works on: offsets inside a longer list, sequences without tokens."""
    g = ops.rng(4)
    n, page, total = len(bad) - 1, 16, 4000
    s = torch.cuda.current_stream()
    i32 = dict(dtype=torch.int32, device="cuda")
    good = torch.tensor([0] + [total * (i + 1) // n for i in range(n)], **i32)
    off = torch.tensor(bad, **i32)
    cache, table = ops.make_cache(g, [total] * n, 2, 64, page)
    zero = torch.zeros(n, **i32)

    def refused(call, *args, **kw):
        call(*args, stream=s, **kw)
        with pytest.raises(P.InvalidInput, match="out of range"):
            gpu.synchronize(s)

    for dtype in (torch.float32, torch.bfloat16):
        q, k, v = (torch.randn(total, 2, 64, device="cuda", generator=g).to(dtype) for _ in range(3))
        for a, b in ((off, good), (good, off)):
            refused(gpu.attention_packed, q, k, v, a, b, torch.empty_like(q), causal=True)
        refused(gpu.attention_packed, q[:, :, :15], k[:, :, :15], v[:, :, :15], off, good, torch.empty_like(q)[:, :, :15])
        refused(gpu.cache_read, cache, k, v, off, zero, table)
        refused(gpu.cache_append, cache, k, v, off, zero, table)
    gpu.synchronize(s)   # reported once each


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("n", [100, 1000])
def test_packed_masked_keys_change_no_bit(gpu, n, d, dtype):
    """Keys that only the last queries see, with scores far above the others', leave the other rows as they were."""
    g = ops.rng(n + d)
    q, k, v = (torch.randn(n, h, d, device="cuda", generator=g).to(DT[dtype]) for h in (4, 2, 2))
    outs = []
    for factor in (1, 1000):
        kk = k.clone()
        kk[n - 3:] *= factor
        outs.append(packed(gpu, q, kk, v, [n], [n], True))
    assert torch.equal(outs[0][:n - 3], outs[1][:n - 3])


# ---------------------------------------------------------------------------
# Packed attention: scores beyond what FP32 resolves
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("n,at", [(40, 5), (40, 17), (700, 0), (700, 334), (700, 339), (700, 350), (700, 699)])
@pytest.mark.parametrize("power", [20, 28, 32, 36, 44, 70])
def test_packed_scores_far_beyond_their_roundings(gpu, power, n, at, d, dtype):
    """Scores near 2^power, of either rounding, whose largest is four times the next: its key's value alone."""
    g = ops.rng(power + at)
    q = torch.zeros(n, 1, d, device="cuda")
    q[:, 0, 0] = (1 + torch.rand(n, device="cuda", generator=g)) * 2.0 ** (power - power // 2)
    k = torch.zeros(n, 1, d, device="cuda")
    k[:, 0, 0] = torch.rand(n, device="cuda", generator=g) * 2.0 ** (power // 2)
    k[at, 0, 0] = (1 + torch.rand(1, device="cuda", generator=g).item()) * 4 * 2.0 ** (power // 2)
    v = torch.randn(n, 1, d, device="cuda", generator=g)
    q, k, v = (x.to(DT[dtype]) for x in (q, k, v))
    for scale in (1.0, 0.7, 0.9):
        out = packed(gpu, q, k, v, [n], [n], scale=scale)
        ref = v[at].double().expand(n, 1, d)
        ops.check(out, ref, ref.abs() * (2 * HALF_STEP[dtype] + 2.0 ** -20) + 1e-30, f"scale {scale}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [40, 700])
@pytest.mark.parametrize("power", [24, 33, 40])
def test_packed_equal_scores_far_beyond_their_roundings(gpu, power, n, dtype):
    """The same key at several places, far above the others: the mean of its values."""
    d, at = 64, [1, 6, 13, 30, n - 1]
    g = ops.rng(power + n)
    q, k = torch.zeros(n, 1, d, device="cuda"), torch.zeros(n, 1, d, device="cuda")
    q[:, 0, 3] = (1 + torch.rand(n, device="cuda", generator=g)) * 2.0 ** power
    k[:, 0, 3] = torch.rand(n, device="cuda", generator=g)
    k[at, 0, 3] = 4.7
    v = torch.randn(n, 1, d, device="cuda", generator=g)
    q, k, v = (x.to(DT[dtype]) for x in (q, k, v))
    for scale in (1.0, 0.7, 0.9):
        out = packed(gpu, q, k, v, [n], [n], scale=scale)
        ref, mag = v[at].double().mean(0).expand(n, 1, d), v[at].double().abs().mean(0).expand(n, 1, d)
        ops.check(out, ref, HALF_STEP[dtype] * ref.abs() + mag * (HALF_STEP[dtype] + 2.0 ** -20) + 1e-30, f"scale {scale}")


# ---------------------------------------------------------------------------
# Single-token attention: pages whose values lie far apart
# ---------------------------------------------------------------------------

def check_cached_relative(out, q, cache, table, lengths, page, dtype):
    """As the other tests' check, but what a small weight may lose is counted relative to the largest product of a
    weight and its V scale: 2^-31 for the one FP16 piece of BF16 calls, 2^-41 for the two of FP32 ones; 2^-133 and
    2^-147 are steps of the smallest numbers."""
    d = q.shape[-1]
    for i, n in enumerate(lengths):
        k, v = ops.cache_values(cache, table, i, n, page)
        ref, mag, prod = ops.attend(q[i:i + 1].double(), k, v, d ** -0.5)
        tol = ops.tolerance(ref, mag, prod, d, n, dtype, 2.0 ** -11 if dtype == "bf16" else 2.0 ** -20) - 1e-30
        rows = table[i, : -(-n // page)].long()
        scales = cache.v_scales[rows].double().repeat_interleave(page, 0)[:n, :, None].expand(-1, -1, d)
        group, heads = q.shape[1] // k.shape[1], []
        for h in range(q.shape[1]):
            w = torch.softmax(k[:, h // group] @ q[i, h].double() * d ** -0.5, 0)
            heads.append((w * scales[:, h // group, 0]).amax())
        most = torch.stack(heads)
        floor = n * 127 * most * (2.0 ** -31 if dtype == "bf16" else 2.0 ** -41)
        tol = tol + floor[None, :, None] + (2.0 ** -133 if dtype == "bf16" else 2.0 ** -147) + n * 2.0 ** -143
        ops.check(out[i:i + 1], ref, tol, f"sequence {i}, length {n}")


def cached(gpu, cache, q, lengths, table):
    s = torch.cuda.current_stream()
    out = torch.full_like(q, 7.0)
    gpu.attention_cached(cache, q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table, out, stream=s)
    gpu.synchronize(s)
    return out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("small", [1e-45, 1e-42, 1e-38, 1e-37, 1e-34, 1e-30])
def test_cached_small_value_scales(gpu, small, d, dtype):
    """Pages of the smallest values, alone and ahead of ordinary ones."""
    g = ops.rng(d)
    lengths, page = [40, 100, 333, 7], 16
    cache, table = ops.make_cache(g, lengths, 2, d, page)
    cache.v_scales[table[0, :3].long()] = small
    cache.v_scales[table[1, 0].long()] = small
    cache.v_scales[table[2, :20].long()] = small
    cache.v_scales[table[3, 0].long()] = small
    q = torch.randn(4, 4, d, device="cuda", generator=g).to(DT[dtype])
    out = cached(gpu, cache, q, lengths, table)
    check_cached_relative(out, q, cache, table, lengths, page, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("power", [8, 12, 20, 27, 40, 60, 90])
def test_cached_large_values_of_little_weight(gpu, power, where, dtype):
    """A page whose values are 2^power times the others' but whose keys score far below: next to nothing."""
    d, page, lengths = 64, 16, [333, 90, 5000]
    g = ops.rng(power)
    cache, table = ops.make_cache(g, lengths, 2, d, page)
    cache.k.clamp_(-30, 30)
    q = (0.5 + torch.rand(3, 4, d, device="cuda", generator=g)).to(DT[dtype])
    for i, n in enumerate(lengths):
        blocks = -(-n // page)
        at = table[i, {"first": 0, "middle": blocks // 2, "last": blocks - 1}[where]].long()
        cache.k[at] = -100
        cache.k_scales[at] = (power * math.log(2) + 40) * 8 / (100 * 0.5 * d)   # scores of -40 - power ln 2 and less
        cache.v_scales[at] = cache.v_scales[at] * 2.0 ** power
    out = cached(gpu, cache, q, lengths, table)
    check_cached_relative(out, q, cache, table, lengths, page, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_cached_value_scales_up_to_the_largest(gpu, dtype):
    """Values near FP32's largest: those of ordinary pages next to them vanish, nothing overflows."""
    d, page, lengths = 64, 16, [200, 40]
    g = ops.rng(50)
    cache, table = ops.make_cache(g, lengths, 2, d, page)
    cache.k.clamp_(-3, 3)
    cache.v.clamp_(-100, 100)
    for i in range(2):
        cache.v_scales[table[i, 1:3].long()] = 3e36
    q = torch.randn(2, 4, d, device="cuda", generator=g).to(DT[dtype])
    out = cached(gpu, cache, q, lengths, table)
    check_cached_relative(out, q, cache, table, lengths, page, dtype)


# ---------------------------------------------------------------------------
# FP32: channels far apart
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("d", [15, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("apart", [16, 22, 28])
def test_packed_fp32_channels_of_different_powers(gpu, n, d, causal, apart):
    """Columns of V up to 2^-apart of the others keep FP32's precision, and so do the products of a small channel of
    q with a large one of k."""
    g = ops.rng(n + apart)
    q, k, v = (torch.randn(n, h, d, device="cuda", generator=g) for h in (4, 2, 2))
    down = torch.exp2(-torch.randint(0, apart + 1, (d,), device="cuda", generator=g).float())
    v *= down
    other = torch.exp2(-torch.randint(0, apart + 1, (d,), device="cuda", generator=g).float())
    q, k = q * other, k / other
    out = packed(gpu, q, k, v, [n], [n], causal)
    ref, tol = ops.packed_reference(q, k, v, [n], [n], causal, d ** -0.5, "f32")
    ops.check(out, ref, tol)


@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("apart", [40, 70])
def test_packed_fp32_channels_too_far_apart(gpu, n, apart):
    """Beyond that a value keeps 2^-50 of its row's largest, twice over two roundings of it and its weight."""
    d = 64
    g = ops.rng(n + apart)
    q, k, v = (torch.randn(n, 2, d, device="cuda", generator=g) for _ in range(3))
    v[..., ::3] *= 2.0 ** -apart
    out = packed(gpu, q, k, v, [n], [n])
    ref, mag, prod = ops.attend(q.double(), k.double(), v.double(), d ** -0.5)
    row = v.abs().amax(-1, keepdim=True).expand(-1, -1, d).double()
    most = ops.attend(q.double(), k.double(), row, d ** -0.5)[0]
    ops.check(out, ref, ops.tolerance(ref, mag, prod, d, n, "f32", 2.0 ** -20) + most * 2.0 ** -49)


@pytest.mark.parametrize("d", [24, 64, 128])
@pytest.mark.parametrize("apart", [16, 22, 28])
def test_cached_fp32_query_channels_of_different_powers(gpu, d, apart):
    """The small channels of a query count where the large ones meet keys of 0."""
    g = ops.rng(apart + d)
    lengths, page = [40, 1000], 16
    cache, table = ops.make_cache(g, lengths, 2, d, page)
    q = torch.randn(2, 4, d, device="cuda", generator=g)
    cache.k[..., :4] = 0
    q[..., 4:] *= 2.0 ** -apart
    cache.k_scales *= 2.0 ** apart
    out = cached(gpu, cache, q, lengths, table)
    check_cached_relative(out, q, cache, table, lengths, page, "f32")


# ---------------------------------------------------------------------------
# Scales and queries whose product passes FP32 while the scores do not
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [40, 700])
@pytest.mark.parametrize("d", [16, 64])
def test_packed_negative_scores_of_large_scales(gpu, n, d, dtype):
    """Every score finite and negative: the least negative one's value."""
    g = ops.rng(n)
    q, k = torch.zeros(n, 1, d, device="cuda"), torch.zeros(n, 1, d, device="cuda")
    q[..., 1] = 2.0 ** 45
    k[..., 1] = -(1 + torch.rand(n, 1, device="cuda", generator=g)) * 2.0 ** -20
    k[n // 2, 0, 1] = -2.0 ** -21
    v = torch.randn(n, 1, d, device="cuda", generator=g)
    q, k, v = (x.to(DT[dtype]) for x in (q, k, v))
    out = packed(gpu, q, k, v, [n], [n], scale=1e30)
    ref = v[n // 2].double().expand(n, 1, d)
    ops.check(out, ref, ref.abs() * (2 * HALF_STEP[dtype] + 2.0 ** -20) + 1e-30)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("power,scale", [(45, 1e30), (90, 1.0), (60, 1e-20)])
def test_cached_negative_scores_of_large_scales(gpu, power, scale, dtype):
    g = ops.rng(power)
    lengths, page, d = [90, 1000], 16, 64
    cache, table = ops.make_cache(g, lengths, 1, d, page)
    cache.k.zero_()
    cache.k[..., 2] = torch.randint(-128, -100, cache.k.shape[:3], device="cuda", generator=g).to(torch.int8)
    cache.k_scales.fill_(2.0 ** (100 - power) / scale)   # scores near -2^107
    at = [(0, 47), (1, 733)]
    for i, t in at:
        cache.k[table[i, t // page].long(), 0, t % page, 2] = -50
    q = torch.zeros(2, 3, d, device="cuda")
    q[..., 2] = 2.0 ** power
    q = q.to(DT[dtype])
    s = torch.cuda.current_stream()
    out = torch.full_like(q, 7.0)
    gpu.attention_cached(cache, q, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table, out, scale=scale, stream=s)
    gpu.synchronize(s)
    for i, t in at:
        row = table[i, t // page].long()
        ref = (cache.v[row, 0, t % page].double() * cache.v_scales[row, 0].double()).expand(3, d)
        ops.check(out[i], ref, ref.abs() * (HALF_STEP[dtype] + (2.0 ** -11 if dtype == "bf16" else 2.0 ** -20)) + 1e-30)


# ---------------------------------------------------------------------------
# Waiting
# ---------------------------------------------------------------------------

def test_waiting_for_a_busy_stream_of_the_callers_leaves_the_handle_usable():
    gpu = P.Gpu(0)
    s = torch.cuda.Stream()
    x = torch.randn(2, 100, device="cuda")
    bad = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    mask = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    gpu.logit_rules(x, torch.empty_like(x), mask=mask, mask_index=bad, stream=s)
    with torch.cuda.stream(s):
        torch.cuda._sleep(400_000_000)   # about 0.2 s
    with pytest.raises(P.GpuError, match="wait limit"):
        gpu.synchronize(s, timeout_ms=5)
    with pytest.raises(P.InvalidInput, match="out of range"):   # still to be reported
        gpu.synchronize(s)
    out = gpu.logit_rules(x, torch.empty_like(x), bias=torch.ones(100, device="cuda"), stream=s)
    gpu.synchronize(s)
    assert torch.equal(out, x + 1)
    gpu.close()


# ---------------------------------------------------------------------------
# Offsets past 32 bits, the smallest scales
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pages_past_32_bits(gpu, dtype):
    """Pages 2^31 and 2^32 bytes into the cache answer as the same ones of a small cache do."""
    page, kv, d, lengths = 128, 8, 128, [700, 129]
    cell = page * kv * d
    pages = 2 ** 32 // cell + 9
    g = ops.rng(60)
    small, table = ops.make_cache(g, lengths, kv, d, page)
    n = small.k.shape[0]
    places = torch.tensor([0, 2 ** 31 // cell - 1, 2 ** 31 // cell, 2 ** 32 // cell - 1, 2 ** 32 // cell, pages - 1] +
                          list(range(7, 7 + n)), device="cuda")[:n]
    big = P.PagedCache(*(torch.empty(pages, *x.shape[1:], dtype=x.dtype, device="cuda")
                         for x in (small.k, small.v, small.k_scales, small.v_scales)))
    for x, y in zip((big.k, big.v, big.k_scales, big.v_scales), (small.k, small.v, small.k_scales, small.v_scales)):
        x[places] = y
    far = torch.where(table >= 0, places[table.clamp_min(0).long()].int(), -1)
    s = torch.cuda.current_stream()
    held = torch.tensor([690, 120], dtype=torch.int32, device="cuda")
    new = [torch.randn(19, kv, d, device="cuda", generator=g).to(DT[dtype]) for _ in range(2)]
    q = torch.randn(2, 16, d, device="cuda", generator=g).to(DT[dtype])
    outs = []
    for cache, where in ((small, table), (big, far)):
        gpu.cache_append(cache, *new, ops.offsets([10, 9]), held, where, stream=s)
        k, v = (torch.empty(sum(lengths), kv, d, dtype=DT[dtype], device="cuda") for _ in range(2))
        gpu.cache_read(cache, k, v, ops.offsets(lengths), torch.zeros_like(held), where, stream=s)
        outs.append([k, v, cached(gpu, cache, q, lengths, where)])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [5, 9])
@pytest.mark.parametrize("d", [15, 64])
def test_packed_strides_past_32_bits(gpu, n, d, dtype):
    """Tokens 2^29 and more values apart."""
    step = 2 ** 29 + 64
    g = ops.rng(n)
    whole = torch.empty((n - 1) * step + 3 * d, dtype=DT[dtype], device="cuda")
    q, k, v = (whole[i * d:].as_strided((n, 1, d), (step, d, 1)) for i in range(3))
    near = [torch.randn(n, 1, d, device="cuda", generator=g).to(DT[dtype]) for _ in range(3)]
    for x, y in zip((q, k, v), near):
        x.copy_(y)
    out = packed(gpu, *near, [n], [n], True)
    far = torch.empty_like(near[0])
    s = torch.cuda.current_stream()
    gpu.attention_packed(q, k, v, ops.offsets([n]), ops.offsets([n]), far, causal=True, stream=s)
    gpu.synchronize(s)
    assert torch.equal(out, far)
    gpu.attention_packed(*near, ops.offsets([n]), ops.offsets([n]), q, causal=True, stream=s)
    gpu.synchronize(s)
    assert torch.equal(out, q) and torch.equal(k, near[1]) and torch.equal(v, near[2])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [40, 700])
def test_the_smallest_scales_weigh_all_keys_alike(gpu, n, dtype):
    g = ops.rng(n)
    d, page = 64, 16
    q, k, v = (torch.randn(n, 2, d, device="cuda", generator=g).to(DT[dtype]) for _ in range(3))
    weight = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -20
    for scale in (2.0 ** -149, 1e-38):
        out = packed(gpu, q, k, v, [n], [n], True, scale=scale)
        zero = torch.zeros_like(q).double()
        ref, mag, prod = ops.attend(zero, zero, v.double(), 1.0, 0)
        ops.check(out, ref, ops.tolerance(ref, mag, prod, d, n, dtype, weight))
        cache, table = ops.make_cache(g, [n], 2, d, page)
        s = torch.cuda.current_stream()
        one = torch.empty_like(q[:1])
        gpu.attention_cached(cache, q[:1], torch.tensor([n], dtype=torch.int32, device="cuda"), table, one, scale=scale, stream=s)
        gpu.synchronize(s)
        kk, vv = ops.cache_values(cache, table, 0, n, page)
        ref, mag, prod = ops.attend(zero[:1], torch.zeros_like(kk), vv, 1.0)
        ops.check(one, ref, ops.tolerance(ref, mag, prod, d, n, dtype, 2.0 ** -11 if dtype == "bf16" else 2.0 ** -20))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_no_numbers_behind_a_sequence_cost_nothing(gpu, d, causal):
    """NaN behind every sequence, in its last tile of keys, does not send its rows to the second computation."""
    g = ops.rng(d)
    lengths, behind = [1990, 1990], 150
    s = torch.cuda.current_stream()
    q, k, v = (torch.randn(sum(lengths) + 2 * behind, h, d, device="cuda", generator=g).bfloat16() for h in (16, 2, 2))
    # Offsets leave a gap behind each sequence, as an allocation with room to grow does.
    first = [0, lengths[0] + behind]
    rows = torch.cat([torch.arange(a, a + n, device="cuda") for a, n in zip(first, lengths)])
    gap = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    gap[rows] = False
    times, outs = [], []
    for fill in (0.0, math.nan):
        k[gap], v[gap] = fill, fill
        one = []
        for a, n in zip(first, lengths):
            off = torch.tensor([a, a + n], dtype=torch.int32, device="cuda")
            out = torch.zeros_like(q)
            for _ in range(3):
                marks = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
                marks[0].record()
                gpu.attention_packed(q, k, v, off, off, out, causal=causal, stream=s)
                marks[1].record()
                gpu.synchronize(s)
            one.append(out[a:a + n])
            times.append(marks[0].elapsed_time(marks[1]))
        outs.append(torch.cat(one))
    assert torch.equal(*outs)
    assert max(times[2:]) < 20 * max(times[:2])   # 84 ms against 0.06 when they did


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_cached_scales_of_either_sign(gpu, dtype):
    """A cache of the caller's own making may hold negative scales."""
    g = ops.rng(70)
    lengths, page, d = [100, 900, 17], 16, 64
    cache, table = ops.make_cache(g, lengths, 2, d, page)
    for x in (cache.k_scales, cache.v_scales):
        x *= torch.where(torch.rand(x.shape, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    cache.v_scales[table[0, :3].long()] = -cache.v_scales[table[0, :3].long()].abs()
    q = torch.randn(3, 4, d, device="cuda", generator=g).to(DT[dtype])
    out = cached(gpu, cache, q, lengths, table)
    for i, n in enumerate(lengths):
        k, v = ops.cache_values(cache, table, i, n, page)
        ref, mag, prod = ops.attend(q[i:i + 1].double(), k, v, d ** -0.5)
        tol = ops.tolerance(ref, mag, prod, d, n, dtype, 2.0 ** -11 if dtype == "bf16" else 2.0 ** -20)
        ops.check(out[i:i + 1], ref, tol + n * 2.0 ** -31 * v.abs().max())
