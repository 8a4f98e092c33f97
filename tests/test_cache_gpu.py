"""The paged 8-bit cache on an MI355X: appending against the definition byte by byte, attention against 64 bits within the error
that its roundings can make (tests/cache_reference.py), and the two together as a decoding program runs them."""
import ctypes
import math
import os

import numpy as np
import pytest
import torch

import cache_reference as ref
from rocmkernels_amd import attention as abi
from rocmkernels_amd import cache as kv

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def noise(seed, *shape):
    return torch.from_numpy(np.random.RandomState(seed).standard_normal(shape).astype(np.float32))


def tables(positions, width, seed=0):
    """cos and sin of rotations by position, both halves their own (no relation between them is assumed)."""
    angle = np.arange(positions)[:, None] * (10000.0 ** (-2.0 * (np.arange(width) % (width // 2)) / width))[None]
    return torch.from_numpy(np.cos(angle).astype(np.float32)), torch.from_numpy(np.sin(angle + 0.01 * seed).astype(np.float32))


def filled_cache(device, pages, size, heads, width, seed, low=-9, high=-5):
    """A cache of random finite e4m3 bytes and scales 2^low .. 2^high."""
    r = np.random.RandomState(seed)

    def cells(*shape):
        b = r.randint(0, 127, shape).astype(np.uint8) | (r.randint(0, 2, shape).astype(np.uint8) << 7)
        return torch.from_numpy(b).view(torch.float8_e4m3fn).to(device)

    scales = torch.from_numpy(np.exp2(r.randint(low, high + 1, (pages, heads, 2))).astype(np.float32)).to(device)
    return kv.KVCache(cells(pages, heads, size // 16, 16, width), cells(pages, heads, size // 16, width, 16), scales)


def batch_of(device, counts, lengths, size, pages, seed, spare=0):
    """starts, lengths and a table of distinct pages in random order; ``spare`` columns beyond what the lengths need."""
    columns = max(1, max((n + size - 1) // size for n in lengths)) + spare
    order = np.random.RandomState(seed).permutation(pages)
    need = [(n + size - 1) // size for n in lengths]
    assert sum(need) <= pages
    table, at = np.zeros((len(counts), columns), np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return [torch.from_numpy(np.asarray(a, np.int32)).to(device) for a in (table, starts, np.asarray(lengths, np.int32))]


def same_bytes(got, want, label):
    """e4m3 bytes, any NaN as good as another."""
    nan = ((got & 0x7f) == 0x7f) & ((want & 0x7f) == 0x7f)
    differ = (got != want) & ~nan
    assert not differ.any(), f"{label}: {int(differ.sum())} bytes differ, first at {np.argwhere(differ)[0]}"


def check_append(cache, k, v, table, starts, lengths, q=None, cos=None, sin=None, label=""):
    want = ref.Pages(cache.keys, cache.values, cache.scales)
    out = None
    if q is not None:
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device=q.device)
    host = lambda t: None if t is None else t.cpu()  # noqa: E731
    turned = ref.append(want, host(k), host(v), table.cpu().numpy(), starts.cpu().numpy(), lengths.cpu().numpy(), host(q), host(cos),
                        host(sin), host(out))
    got_q = kv.append(cache, k, v, table, starts, lengths, q=q, cos=cos, sin=sin, out_q=out)
    torch.cuda.synchronize()
    got = ref.Pages(cache.keys, cache.values, cache.scales)
    assert np.array_equal(got.scales, want.scales, equal_nan=True), f"{label}: scales"
    same_bytes(got.k, want.k, f"{label}: keys")
    same_bytes(got.v, want.v, f"{label}: values")
    if q is None:
        assert got_q is None
    else:
        assert torch.equal(got_q.cpu().nan_to_num(123.0), torch.from_numpy(turned).to(q.dtype).nan_to_num(123.0)), f"{label}: queries"


def check_attention(cache, q, table, starts, lengths, label="", **how):
    output = torch.full(q.shape, 7.0, dtype=q.dtype, device=q.device)
    lse = torch.full(q.shape[:2] + (2,), 7.0, device=q.device)
    kv.attention(cache, q, table, starts, lengths, output=output, lse=lse, **how)
    torch.cuda.synchronize()
    pages = ref.Pages(cache.keys, cache.values, cache.scales)
    out, stats, tol, lse_tol = ref.attention(pages, q.cpu(), table.cpu().numpy(), starts.cpu().numpy(), lengths.cpu().numpy(), **how)
    got, got_lse = output.double().cpu().numpy(), lse.double().cpu().numpy()
    mine = np.zeros(q.shape[0], bool)
    for _, row, count, _ in ref.spans(starts.cpu().numpy(), lengths.cpu().numpy(), q.shape[0]):
        mine[row:row + count] = True
    assert (got[~mine] == 7.0).all() and (got_lse[~mine] == 7.0).all(), f"{label}: rows of no sequence were written"
    got, got_lse, out, stats, tol, lse_tol = (a[mine] for a in (got, got_lse, out, stats, tol, lse_tol))
    assert np.array_equal(np.isnan(got), np.isnan(out)), f"{label}: NaN in {np.isnan(got).sum()} outputs, {np.isnan(out).sum()} expected"
    # Past the type's largest value by half a step, nearest-even rounding gives infinity; within the bound of that either is right.
    edge = torch.finfo(q.dtype).max * (1 + torch.finfo(q.dtype).eps / 4)
    over, near = np.abs(out) - tol >= edge, np.abs(out) + tol >= edge
    assert np.array_equal(got[over], np.copysign(np.inf, out[over])), f"{label}: overflow"
    fine = np.isfinite(out) & ~near
    worst = (np.abs(got - out)[fine] / np.maximum(tol[fine], 1e-300)).max(initial=0.0)
    assert worst <= 1.0, f"{label}: output off by {worst:.2f} of the bound"
    empty = np.isneginf(stats[..., 0])
    assert np.isneginf(got_lse[..., 0][empty]).all() and (got_lse[..., 1][empty] == 0).all() and (got[empty] == 0).all(), label
    known = np.isfinite(stats).all(-1)
    with np.errstate(invalid="ignore"):
        worst = (np.abs(got_lse - stats)[known] / np.maximum(lse_tol[known], 1e-300)).max(initial=0.0)
    assert worst <= 1.0, f"{label}: lse off by {worst:.2f} of the bound"


# ---- append -------------------------------------------------------------------------------------------------------
APPENDS = [
    # counts, lengths: one token; a page's first and last slot; several pages; uneven; empty sequences between others
    ([1], [1]), ([1], [16]), ([1], [17]), ([3], [130]), ([1, 1, 1, 1, 1], [1, 16, 33, 64, 129]),
    ([0, 5, 0, 1, 37, 0], [20, 5, 0, 100, 90, 3]), ([150], [150]), ([70, 9], [200, 9]), ([16, 32, 48], [64, 32, 129]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [32, 64, 128])
@pytest.mark.parametrize("size", [16, 48, 64, 128])
def test_append(device, dtype, width, size):
    for n, (counts, lengths) in enumerate(APPENDS):
        heads, group, pages = 3, (1, 4, 2)[n % 3], 24
        cache = filled_cache(device, pages, size, heads, width, 10 + n)
        table, starts, ends = batch_of(device, counts, lengths, size, pages, n, spare=n % 2)
        tokens = sum(counts) + n % 2  # sometimes a row behind the last sequence
        k, v, q = (noise(100 * n + i, tokens, h, width).to(DTYPES[dtype]).to(device) for i, h in enumerate((heads, heads, heads * group)))
        cos, sin = (t.to(device) for t in tables(max(lengths) + 1, width, n))
        check_append(cache, k, v, table, starts, ends, q, cos, sin, f"{counts} {lengths}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_without_rotation_or_queries(device, dtype):
    cache = filled_cache(device, 12, 32, 2, 64, 3)
    table, starts, ends = batch_of(device, [5, 40], [37, 40], 32, 12, 3)
    k, v = (noise(i, 45, 2, 64).to(DTYPES[dtype]).to(device) for i in range(2))
    check_append(cache, k, v, table, starts, ends, label="no rotation")
    cos, sin = (t.to(device) for t in tables(64, 64))
    check_append(cache, k, v, table, starts, ends, cos=cos, sin=sin, label="no queries")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [32, 128])
@pytest.mark.parametrize("count", [1, 30])
def test_append_strided_rows(device, dtype, width, count):
    """Rows cut out of a fused projection, at an odd offset that no 128-bit access fits."""
    heads, group, tokens = 2, 3, 2 * count
    for offset, extra in ((0, 0), (8, 8), (1, 3)):
        across = (heads * group + 2 * heads) * width + offset + extra
        flat = noise(5, tokens, across).to(DTYPES[dtype]).to(device)
        parts = flat[:, offset:offset + (heads * group + 2 * heads) * width].unflatten(1, (-1, width))
        q, k, v = parts[:, :heads * group], parts[:, heads * group:heads * (group + 1)], parts[:, heads * (group + 1):]
        cache = filled_cache(device, 8, 64, heads, width, 6)
        table, starts, ends = batch_of(device, [count, count], [count + 9, count], 64, 8, 7)
        cos, sin = (t.to(device) for t in tables(count + 9, width + offset))
        check_append(cache, k, v, table, starts, ends, q, cos[:, :width], sin[:, :width], f"offset {offset}")


def test_append_rotates_queries_in_place(device):
    cache = filled_cache(device, 4, 64, 2, 64, 8)
    table, starts, ends = batch_of(device, [6], [50], 64, 4, 8)
    k, v, q = (noise(i, 6, h, 64).to(device) for i, h in enumerate((2, 2, 4)))
    cos, sin = (t.to(device) for t in tables(64, 64))
    apart = kv.append(cache, k, v, table, starts, ends, q=q, cos=cos, sin=sin)
    assert kv.append(cache, k, v, table, starts, ends, q=q, cos=cos, sin=sin, out_q=q) is q
    assert torch.equal(q, apart)


@pytest.mark.parametrize("steps", [1, 7, 20])
def test_append_grows_scales(device, steps):
    """Tokens one by one (and in small groups), each larger than the ones before: earlier rows are requantised every time, down into
    e4m3's subnormals and to zero."""
    width, heads, size = 64, 2, 32
    cache = kv.KVCache.empty(3, size, heads, width, device)
    at = 0
    for step in range(steps):
        count = 1 + step % 3
        at += count
        table, starts, ends = batch_of(device, [count], [at], size, 3, 1)
        big = 1.7 ** step * (1 if step % 5 else 1000)
        k, v = noise(step, count, heads, width).to(device) * big, noise(50 + step, count, heads, width).to(device) / big
        check_append(cache, k, v, table, starts, ends, label=f"step {step}")


def test_append_again_after_rejection(device):
    """Drafted tokens are appended, some rejected, and others appended in their place."""
    cache = filled_cache(device, 6, 16, 2, 32, 4)
    cos, sin = (t.to(device) for t in tables(64, 32))
    for step, (count, length) in enumerate([(5, 22), (4, 20), (1, 18), (9, 26), (9, 26)]):
        table, starts, ends = batch_of(device, [count], [length], 16, 6, 2, spare=2)
        k, v, q = (noise(10 * step + i, count, 2, 32).to(torch.bfloat16).to(device) for i in range(3))
        check_append(cache, k, v, table[:, :4], starts, ends, q, cos, sin, f"step {step}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 20])
def test_append_odd_values(device, dtype, count):
    """Zeros, subnormals, the type's largest values, infinities and NaN, and scales of a page that hold anything."""
    width, heads, size = 32, 4, 16
    cache = filled_cache(device, 8, size, heads, width, 9)
    cache.scales[:, 0] = 0.0
    cache.scales[:, 1] = float("nan")
    cache.scales[:, 2] = 2.0 ** -120
    table, starts, ends = batch_of(device, [count], [count + 5], size, 8, 9)
    info = torch.finfo(DTYPES[dtype])
    k, v = noise(1, count, heads, width).to(DTYPES[dtype]), noise(2, count, heads, width).to(DTYPES[dtype])
    k[:, 0] = 0.0
    k[0, 1, :4] = torch.tensor([math.inf, -math.inf, math.nan, 1.0])
    k[-1, 2, :3] = torch.tensor([info.max, -info.max, info.tiny])
    v[:, 0] = info.tiny / 4
    v[-1, 1] = math.nan
    v[0, 2, 5] = info.max
    v[0, 3] = math.inf
    check_append(cache, k.to(device), v.to(device), table, starts, ends, label="odd values")


def test_append_values_next_to_a_step(device):
    """Every e4m3 value, the midpoints between neighbours and the floats next to them round as the definition says."""
    values = np.sort(ref.from_e4m3(np.arange(0x7f, dtype=np.uint8)))
    mid = ((values[1:] + values[:-1]) / 2).astype(np.float32)
    x = np.concatenate([values.astype(np.float32), mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1000))])
    x = np.concatenate([x, -x])
    x = np.pad(x, (0, -len(x) % 128), constant_values=448.0).reshape(-1, 1, 128)
    tokens = len(x)
    cache = kv.KVCache.empty(4, 16, 1, 128, device)
    table, starts, ends = batch_of(device, [tokens], [tokens], 16, 4, 5)
    x = torch.from_numpy(x).to(device)
    check_append(cache, x, x, table, starts, ends, label="steps")


def test_append_leaves_out_what_has_no_place(device):
    """Bad page ids, positions before 0, behind the table and behind cos and sin, rows behind the last sequence."""
    size, heads, width = 16, 2, 64
    cache = filled_cache(device, 6, size, heads, width, 11)
    table = torch.tensor([[0, -1, 1], [6, 2, 1 << 30], [3, 4, 5], [-(1 << 31), 0, 0]], dtype=torch.int32, device=device)
    # 40 rows over three pages (the second bad); 20 rows up to position 37; 9 rows for 4 keys; 5 rows, the last 3 behind the table
    for counts, lengths, positions in (([40, 20, 9, 0], [40, 38, 4, 0], 100), ([0, 0, 5, 0], [0, 0, 51, 0], 100), ([40, 0, 40, 2], [40, 0, 45, 2], 21)):
        starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=device)
        ends = torch.tensor(lengths, dtype=torch.int32, device=device)
        tokens = sum(counts) + 4
        k, v, q = (noise(i, tokens, heads, width).to(torch.float16).to(device) for i in range(3))
        cos, sin = (t.to(device) for t in tables(positions, width))
        check_append(cache, k, v, table, starts, ends, q, cos, sin, f"{counts} {lengths}")


# ---- attention ----------------------------------------------------------------------------------------------------
FORWARDS = [
    # counts, lengths
    ([1], [1]), ([1], [15]), ([1], [64]), ([1], [65]), ([1], [700]),
    ([1, 1, 1, 1, 1, 1], [1, 17, 63, 64, 300, 129]), ([0, 3, 0, 1, 20, 0], [9, 3, 0, 70, 33, 40]), ([5, 4], [131, 66]), ([90], [90]),
    ([33, 2], [150, 40]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [32, 64, 128])
@pytest.mark.parametrize("size,group", [(16, 1), (48, 4), (64, 3), (128, 8)])
def test_attention(device, dtype, width, size, group):
    for n, (counts, lengths) in enumerate(FORWARDS):
        heads, pages = 2, 64
        cache = filled_cache(device, pages, size, heads, width, 20 + n)
        table, starts, ends = batch_of(device, counts, lengths, size, pages, n, spare=n % 3)
        q = noise(n, sum(counts) + n % 2, heads * group, width).to(DTYPES[dtype]).to(device)
        check_attention(cache, q, table, starts, ends, f"{counts} {lengths}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal,radius", [(True, 0), (True, 40), (False, -1), (False, 25), (True, 1 << 30), (False, (1 << 31) - 1)])
def test_attention_masks(device, dtype, causal, radius):
    for counts, lengths in (([1, 1], [300, 77]), ([40], [130]), ([7, 70], [200, 100])):
        cache = filled_cache(device, 40, 32, 2, 64, 31)
        table, starts, ends = batch_of(device, counts, lengths, 32, 40, 3, spare=1)
        q = noise(2, sum(counts), 6, 64).to(DTYPES[dtype]).to(device)
        check_attention(cache, q, table, starts, ends, f"{counts} {lengths}", causal=causal, radius=radius)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_long_axis_is_split_and_joined(device, dtype):
    """Few rows over many keys: chunks of the key axis, uneven ends, sequences of one chunk beside others."""
    for width, counts, lengths in ((128, [1], [5000]), (32, [1, 1, 2], [4097, 30, 2100]), (64, [1, 60], [3000, 1500])):
        pages = sum((n + 63) // 64 for n in lengths) + 2
        cache = filled_cache(device, pages, 64, 1, width, 41)
        table, starts, ends = batch_of(device, counts, lengths, 64, pages, 4)
        q = noise(3, sum(counts), 5, width).to(DTYPES[dtype]).to(device)
        check_attention(cache, q, table, starts, ends, f"{counts} {lengths}")
        check_attention(cache, q, table, starts, ends, f"{counts} {lengths} window", radius=1111)
        check_attention(cache, q, table, starts, ends, f"{counts} {lengths} bounded", max_keys=max(lengths))
        check_attention(cache, q, table, starts, ends, f"{counts} {lengths} cut", max_keys=1000)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_many_heads_in_a_group(device, dtype):
    cache = filled_cache(device, 12, 64, 1, 64, 42)
    table, starts, ends = batch_of(device, [1, 3], [200, 130], 64, 12, 4)
    for group in (17, 32, 71):
        q = noise(3, 4, group, 64).to(DTYPES[dtype]).to(device)
        check_attention(cache, q, table, starts, ends, f"group {group}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [32, 128])
def test_attention_strided_rows(device, dtype, width):
    for offset, extra in ((0, 0), (8, 16), (3, 2)):
        flat = noise(5, 7, 4 * width + offset + extra).to(DTYPES[dtype]).to(device)
        q = flat[:, offset:offset + 4 * width].unflatten(1, (4, width))
        cache = filled_cache(device, 16, 16, 2, width, 43)
        table, starts, ends = batch_of(device, [3, 4], [90, 100], 16, 16, 6)
        wide = torch.full((7, 4 * width + offset + extra), 7.0, dtype=q.dtype, device=device)
        output = wide[:, offset:offset + 4 * width].unflatten(1, (4, width))
        got, lse = kv.attention(cache, q, table, starts, ends, output=output)
        want, want_lse = kv.attention(cache, q.contiguous(), table, starts, ends)
        assert got is output and torch.equal(got, want) and torch.equal(lse, want_lse)
        assert (wide[:, :offset] == 7).all() and (wide[:, offset + 4 * width:] == 7).all()
        check_attention(cache, q, table, starts, ends, f"offset {offset}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_scales_far_apart(device, dtype):
    """Pages whose scales differ by up to 2^60 beside each other, and scores that make any of them the one that counts."""
    for low, high in ((-60, 0), (-30, 30), (-100, -90), (-12, -2)):
        cache = filled_cache(device, 20, 16, 2, 64, 44, low, high)
        cache.scales[..., 0] = 2.0 ** -7  # keys of one size: scores up to some dozens
        table, starts, ends = batch_of(device, [2, 1], [150, 100], 16, 20, 6)
        q = (0.2 * noise(3, 3, 4, 64)).to(DTYPES[dtype]).to(device)
        check_attention(cache, q, table, starts, ends, f"2^{low}..2^{high}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_zero_keys_and_tiny_queries(device, dtype):
    cache = kv.KVCache.empty(4, 32, 2, 64, device)
    table, starts, ends = batch_of(device, [2], [70], 32, 4, 6)
    q = noise(3, 2, 4, 64).to(DTYPES[dtype]).to(device)
    check_attention(cache, q, table, starts, ends, "empty cache")
    cache = filled_cache(device, 4, 32, 2, 64, 45)
    check_attention(cache, q * 0, table, starts, ends, "zero queries")
    check_attention(cache, q * torch.finfo(q.dtype).tiny, table, starts, ends, "tiny queries")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_over_many_keys_of_no_value(device, dtype, rows):
    """V all zero (the smallest scale there is) over 65536 keys whose scores rise by just less than what moves the reference: sums of
    weights over 2^-100 stay in range, and lse is exact."""
    size, length, width = 128, 65536, 32
    cache = kv.KVCache.empty(length // size, size, 1, width, device)
    cache.scales[..., 0] = 1.0
    position = torch.arange(length, device=device)
    low = (position % 1024 < 256).view(-1, 1, size // 16, 16)
    cache.keys.view(torch.uint8).view(-1, 1, size // 16, 16, width)[..., 0] = torch.where(low, 0xb8, 0).to(torch.uint8)  # -1 or 0
    table = torch.arange(length // size, dtype=torch.int32, device=device)[None]
    starts, ends = (torch.tensor(t, dtype=torch.int32, device=device) for t in ([0, rows], [length]))
    q = torch.zeros((rows, 1, width), dtype=DTYPES[dtype], device=device)
    q[..., 0] = 30.5  # scores of 0 and -30.5 / sqrt(32) = -5.39, that is -7.78 in the exponent of 2
    check_attention(cache, q, table, starts, ends, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [32, 64])
def test_attention_hidden_keys_may_hold_anything(device, dtype, width):
    """NaN in K, V and their scales where a row does not look: behind the end, in front of the window, behind its own position."""
    size, heads = 32, 2
    nan = torch.full((), 0x7f, dtype=torch.uint8)
    for counts, lengths, radius in (([1, 1], [70, 33], -1), ([6], [50], -1), ([1], [200], 20), ([40], [100], 30)):
        cache = filled_cache(device, 16, size, heads, width, 46)
        table, starts, ends = batch_of(device, counts, lengths, size, 16, 8, spare=1)
        host = table.cpu().numpy()
        kb, vb = cache.keys.view(torch.uint8), cache.values.view(torch.uint8)
        for b, n in enumerate(lengths):
            page, slot = int(host[b, (n - 1) // size]), (n - 1) % size
            for s in range(slot + 1, size):
                kb[page, :, s // 16, s % 16] = nan
                vb[page, :, s // 16, :, s % 16] = nan
        used = set(int(host[b, p]) for b, n in enumerate(lengths) for p in range((n + size - 1) // size))
        for page in set(range(16)) - used:
            cache.scales[page] = math.nan
            kb[page] = nan
            vb[page] = nan
        q = noise(3, sum(counts), heads * 2, width).to(DTYPES[dtype]).to(device)
        check_attention(cache, q, table, starts, ends, f"behind the end {counts}", radius=radius)
        # A key of NaN in the middle of the new rows: rows before it (and far behind it) do not see it, the others do.
        if counts[0] > 1:
            at = lengths[0] - counts[0] // 2
            page, slot = int(host[0, at // size]), at % size
            vb[page, 0, slot // 16, :5, slot % 16] = nan
            check_attention(cache, q, table, starts, ends, f"NaN in V {counts}", radius=radius)
            kb[page, 1, slot // 16, slot % 16, 3] = nan
            check_attention(cache, q, table, starts, ends, f"NaN in K {counts}", radius=radius)
        if radius >= 0:
            page, slot = int(host[0, 0]), 3
            kb[page, :, 0, slot] = nan
            vb[page, :, 0, :, slot] = nan
            check_attention(cache, q, table, starts, ends, f"NaN in front of the window {counts}", radius=radius)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [1, 2])
def test_attention_nan_values_reach_the_rows_that_see_them(device, dtype, group):
    """Prompts of more than one row tile: for a key among the new rows, some waves of a tile see every key of a step and others do
    not; each row that sees the NaN has it, also rows of later tiles, for which no key of that step is hidden."""
    for width, size in ((32, 16), (64, 64), (128, 64)):
        heads, count, length = 2, 200, 230
        cache = filled_cache(device, 12 if size > 16 else 20, size, heads, width, 71)
        table, starts, ends = batch_of(device, [count], [length], size, cache.pages, 8)
        host, vb = table.cpu().numpy(), cache.values.view(torch.uint8)
        for position, head, feature in ((3, 0, 1), (35, 1, 2), (100, 0, width - 1), (140, 1, 7), (229, 0, 9)):
            page, slot = int(host[0, position // size]), position % size
            vb[page, head, slot // 16, feature, slot % 16] = 0xff
        q = noise(3, count, heads * group, width).to(DTYPES[dtype]).to(device)
        check_attention(cache, q, table, starts, ends, f"width {width}")
        check_attention(cache, q, table, starts, ends, f"width {width} window", radius=50)


@pytest.mark.parametrize("batch", [65, 300, 5000])
def test_many_sequences(device, batch):
    """More sequences than a round of the search tests, some without rows, some with a few."""
    r = np.random.RandomState(batch)
    counts = r.choice([0, 1, 1, 1, 2], batch)
    if batch == 300:
        counts[::37] = 40  # prompts among them
    lengths = counts + r.randint(0, 40, batch)
    size, heads, width = 16, 1, 32
    pages = int(((lengths + size - 1) // size).sum()) + 2
    cache = filled_cache(device, pages, size, heads, width, 72)
    table, starts, ends = batch_of(device, list(counts), list(lengths), size, pages, 9)
    tokens = int(counts.sum()) + 3
    k, v, q = (noise(i, tokens, heads, width).to(torch.float16).to(device) for i in range(3))
    cos, sin = (t.to(device) for t in tables(100, width))
    check_append(cache, k, v, table, starts, ends, q, cos, sin, f"batch {batch}")
    check_attention(cache, q, table, starts, ends, f"batch {batch}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width,size", [(128, 64), (64, 48), (32, 16)])
def test_mixed_batch(device, dtype, width, size):
    """A chunk of a prompt, single tokens and drafts over long and short contexts in one call: large and small tiles, each cut into
    chunks."""
    counts, lengths = [1, 150, 0, 1, 4, 70, 1], [2500, 2600, 100, 1, 40, 70, 900]
    heads, group = 2, 4
    pages = sum((n + size - 1) // size for n in lengths) + 1
    cache = filled_cache(device, pages, size, heads, width, 73)
    table, starts, ends = batch_of(device, counts, lengths, size, pages, 9)
    q = noise(3, sum(counts) + 1, heads * group, width).to(DTYPES[dtype]).to(device)
    assert kv.workspace(cache, q, table).numel() > 0
    check_attention(cache, q, table, starts, ends, "mixed")
    check_attention(cache, q, table, starts, ends, "mixed window", radius=700)


# Batches whose large tiles two teams of waves share (tests/cpp/cache_plan_check.cpp holds the plan to it): heads, group, counts,
# lengths, masks. One prompt in one chunk of an odd and an even number of steps, and in two chunks; prompts beside each other, one of
# them short and one without rows; a prompt beside single tokens.
TEAMS = [
    (13, 5, [130], [681], [{"radius": 500}, {"causal": False, "radius": 260}]),
    (13, 5, [130], [2200], [{}]),
    (13, 5, [100, 60, 0, 90], [700, 60, 30, 513], [{}]),
    (16, 5, [150] + [1] * 10, [900, 1, 64, 65, 300, 512, 513, 577, 640, 899, 20], [{}, {"radius": 520}]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width,size", [(32, 64), (64, 48), (128, 16)])
def test_attention_by_two_teams(device, dtype, width, size):
    for n, (heads, group, counts, lengths, masks) in enumerate(TEAMS):
        pages = sum((m + size - 1) // size for m in lengths) + 1
        cache = filled_cache(device, pages, size, heads, width, 81 + n)
        table, starts, ends = batch_of(device, counts, lengths, size, pages, 10 + n)
        q = noise(4 + n, sum(counts) + 1, heads * group, width).to(DTYPES[dtype]).to(device)
        for how in masks:
            check_attention(cache, q, table, starts, ends, f"{counts} {lengths} {how}", **how)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width,size", [(32, 32), (64, 64), (128, 64)])
def test_attention_by_two_teams_at_the_edges(device, dtype, width, size):
    """Sequences far shorter than the table allows (no step for one team, or for both), rows without keys, pages that are not there,
    and NaN in V at positions of either team's steps; twice the same bits."""
    heads, group, count = 13, 5, 130
    pages = (1000 + size - 1) // size + 1
    q = noise(4, count, heads * group, width).to(DTYPES[dtype]).to(device)
    for length in (0, 1, 64, 100, 129):
        cache = filled_cache(device, pages, size, heads, width, 91)
        table, starts, ends = batch_of(device, [count], [1000], size, pages, 11)
        ends[:] = length
        check_attention(cache, q, table, starts, ends, f"length {length}", causal=True)
        check_attention(cache, q, table, starts, ends, f"length {length}, all", causal=False)
    cache = filled_cache(device, pages, size, heads, width, 92)
    table, starts, ends = batch_of(device, [count], [1000], size, pages, 12)
    host, vb = table.cpu().numpy().copy(), cache.values.view(torch.uint8)
    for position, head, feature in ((3, 0, 1), (70, 1, 2), (140, 3, width - 1), (880, 4, 7), (930, 5, 0), (999, 12, 9)):
        vb[int(host[0, position // size]), head, position % size // 16, feature, position % 16] = 0x7f
    check_attention(cache, q, table, starts, ends, "NaN in V")
    check_attention(cache, q, table, starts, ends, "NaN in V, window", radius=500)
    table[0, 1] = -1
    table[0, 400 // size] = pages
    table[0, 999 // size] = -7
    check_attention(cache, q, table, starts, ends, "pages that are not there")
    first, second = (kv.attention(cache, q, table, starts, ends) for _ in range(2))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(first, second))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_nan_and_infinite_queries_stay_in_their_row(device, dtype):
    cache = filled_cache(device, 8, 64, 2, 64, 47)
    table, starts, ends = batch_of(device, [4], [140], 64, 8, 8)
    q = noise(3, 4, 6, 64).to(DTYPES[dtype])
    q[1, 2, 7] = math.nan
    q[2, 5, 9] = math.inf
    output, lse = kv.attention(cache, q.to(device), table, starts, ends)
    bad = torch.zeros(4, 6, dtype=torch.bool)
    bad[1, 2] = bad[2, 5] = True
    assert torch.equal(output.isnan().all(-1).cpu(), bad) and torch.equal(output.isnan().any(-1).cpu(), bad)
    assert torch.equal(lse.isnan().all(-1).cpu(), bad)
    q[1, 2, 7] = q[2, 5, 9] = 0.0
    clean, _ = kv.attention(cache, q.to(device), table, starts, ends)
    assert torch.equal(clean[~bad.to(device)], output[~bad.to(device)])


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_rows_without_keys_and_bad_pages(device, dtype):
    cache = filled_cache(device, 6, 16, 2, 32, 48)
    table = torch.tensor([[0, -1, 1, 2], [6, 7, 1 << 30, -5], [3, 4, 5, 0], [0, 0, 0, 0]], dtype=torch.int32, device=device)
    for counts, lengths in (([3, 2, 9, 1], [60, 50, 4, 0]), ([1, 1, 1, 1], [20, 64, 64, 0]), ([40, 1, 30, 0], [64, 3, 20, 9]),
                            ([2, 2, 2, 2], [500, -7, 1 << 30, 64])):
        starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=device)
        ends = torch.tensor(lengths, dtype=torch.int32, device=device)
        q = noise(3, sum(counts) + 2, 4, 32).to(DTYPES[dtype]).to(device)
        for how in ({}, {"causal": False}, {"radius": 5}):
            if max(lengths) > 64 and how:
                continue
            check_attention(cache, q, table, starts, ends, f"{counts} {lengths} {how}", **how)


def test_attention_reads_beyond_32_bits(device):
    """A cache whose later pages lie past 2^32 bytes, appended to and read there."""
    heads, width, size = 8, 128, 128
    pages = (1 << 32) // (heads * width * size) + 40
    keys = torch.zeros((pages, heads, 8, 16, width), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    values = torch.zeros((pages, heads, 8, width, 16), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    cache = kv.KVCache(keys, values, torch.zeros((pages, heads, 2), device=device))
    table = torch.tensor([[pages - 1, 3, pages - 7], [1, pages - 2, 0]], dtype=torch.int32, device=device)
    starts = torch.tensor([0, 300, 420], dtype=torch.int32, device=device)
    ends = torch.tensor([300, 120], dtype=torch.int32, device=device)
    k, v, q = (noise(i, 420, heads, width).to(torch.bfloat16).to(device) for i in range(3))
    kv.append(cache, k, v, table, starts, ends)
    output, lse = kv.attention(cache, q, table, starts, ends)
    near = kv.KVCache.empty(6, size, heads, width, device)
    low = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=device)
    kv.append(near, k, v, low, starts, ends)
    want, want_lse = kv.attention(near, q, low, starts, ends)
    assert torch.equal(output, want) and torch.equal(lse, want_lse)
    assert torch.equal(cache.keys[pages - 7].view(torch.uint8), near.keys[2].view(torch.uint8))
    assert torch.equal(cache.values[pages - 1].view(torch.uint8), near.values[0].view(torch.uint8))


# ---- together -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_prompt_then_tokens_as_a_program_runs_them(device, dtype):
    """Two sequences: prompts in one call, drafts, single tokens, a late third sequence; every step's attention against 64 bits and
    the cache against the definition."""
    heads, group, width, size = 2, 2, 32, 16
    cache = kv.KVCache.empty(40, size, heads, width, device)
    cos, sin = (t.to(device) for t in tables(160, width))
    table = torch.from_numpy(np.random.RandomState(3).permutation(40)[:30].reshape(3, 10).astype(np.int32)).to(device)
    lengths = np.zeros(3, int)
    for step, counts in enumerate([(37, 50, 0), (1, 1, 0), (4, 1, 0), (1, 1, 61), (1, 1, 1), (1, 1, 1)]):
        lengths += counts
        if step == 3:
            lengths[0] -= 2  # two of the four drafted tokens were rejected
        tokens = sum(counts)
        starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=device)
        ends = torch.tensor(lengths, dtype=torch.int32, device=device)
        k, v, q = (noise(10 * step + i, tokens, n, width).to(DTYPES[dtype]).to(device) for i, n in enumerate((heads, heads, heads * group)))
        check_append(cache, k, v, table, starts, ends, q, cos, sin, f"step {step}")
        turned = kv.append(cache, k, v, table, starts, ends, q=q, cos=cos, sin=sin)
        check_attention(cache, turned, table, starts, ends, f"step {step}")


def test_one_call_or_many_give_the_same_rows(device):
    """A prompt in one call equals its last rows asked for alone, whatever launch shape each takes: twice the bound of one."""
    cache = filled_cache(device, 20, 64, 4, 128, 51)
    q = noise(3, 700, 8, 128).to(torch.float16).to(device)
    table, starts, ends = batch_of(device, [700], [1000], 64, 20, 5)
    whole, whole_lse = (t.double().cpu().numpy() for t in kv.attention(cache, q, table, starts, ends))
    pages = ref.Pages(cache.keys, cache.values, cache.scales)
    for count in (1, 3, 9, 40):
        some = torch.tensor([0, count], dtype=torch.int32, device=device)
        part, part_lse = kv.attention(cache, q[700 - count:], table, some, ends)
        _, _, tol, lse_tol = ref.attention(pages, q[700 - count:].cpu(), table.cpu().numpy(), [0, count], [1000])
        assert (np.abs(part.double().cpu().numpy() - whole[700 - count:]) <= 2 * tol).all()
        assert (np.abs(part_lse.double().cpu().numpy() - whole_lse[700 - count:]) <= 2 * lse_tol).all()


def test_graph_of_a_decoding_step(device):
    """A step captured once and replayed while the program moves lengths, tokens and pages on: every replay against eager calls."""
    heads, group, width, size, batch = 2, 4, 64, 16, 5
    eager, graphed = (kv.KVCache.empty(100, size, heads, width, device) for _ in range(2))
    cos, sin = (t.to(device) for t in tables(400, width))
    table = torch.from_numpy(np.random.RandomState(3).permutation(100).reshape(batch, 20).astype(np.int32)).to(device)
    starts = torch.arange(batch + 1, dtype=torch.int32, device=device)
    lengths = torch.tensor([1, 15, 16, 200, 64], dtype=torch.int32, device=device)
    k, v, q = (torch.empty((batch, n, width), dtype=torch.bfloat16, device=device) for n in (heads, heads, heads * group))
    out_q, output = torch.empty_like(q), torch.empty_like(q)
    lse = torch.empty((batch, heads * group, 2), device=device)
    workspace = kv.workspace(graphed, q, table)

    def step(cache, stream=None):
        kv.append(cache, k, v, table, starts, lengths, q=q, cos=cos, sin=sin, out_q=out_q)
        kv.attention(cache, out_q, table, starts, lengths, output=output, lse=lse, workspace=workspace)

    k.fill_(1), v.fill_(1), q.fill_(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graphed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(graphed)
    graphed.scales.zero_(), graphed.keys.view(torch.uint8).zero_(), graphed.values.view(torch.uint8).zero_()
    for replay in range(4):
        for i, t in enumerate((k, v, q)):
            t.copy_(noise(10 * replay + i, *t.shape))
        step(eager)
        torch.cuda.synchronize()
        want = [t.clone() for t in (out_q, output, lse)]
        for t in (out_q, output, lse):
            t.fill_(math.nan)
        workspace.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        for got, t in zip((out_q, output, lse), want):
            assert torch.equal(got, t), f"replay {replay}"
        assert torch.equal(graphed.keys.view(torch.uint8), eager.keys.view(torch.uint8)), f"replay {replay}"
        assert torch.equal(graphed.values.view(torch.uint8), eager.values.view(torch.uint8)), f"replay {replay}"
        assert torch.equal(graphed.scales, eager.scales), f"replay {replay}"
        lengths += 1


def test_two_streams_with_a_workspace_each(device):
    cases = []
    for i in range(2):
        cache = filled_cache(device, 200, 64, 2, 128, 60 + i)
        table, starts, ends = batch_of(device, [1, 2], [6000, 4000], 64, 200, i)
        q = noise(70 + i, 3, 8, 128).to(torch.float16).to(device)
        cases.append((cache, q, table, starts, ends, torch.cuda.Stream(), kv.attention(cache, q, table, starts, ends)))
    torch.cuda.synchronize()
    results = []
    for _ in range(4):
        for cache, q, table, starts, ends, stream, want in cases:
            results.append((kv.attention(cache, q, table, starts, ends, stream=stream), want))
    torch.cuda.synchronize()
    for got, want in results:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_results_repeat_bit_for_bit(device):
    cache = filled_cache(device, 300, 64, 2, 64, 61)
    table, starts, ends = batch_of(device, [1, 70, 3], [9000, 5000, 2000], 64, 300, 2)
    q = noise(71, 74, 4, 64).to(device)
    first = kv.attention(cache, q, table, starts, ends)
    for _ in range(5):
        again = kv.attention(cache, q, table, starts, ends)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


def test_cpp_wrappers_match_c_entry_points(device):
    path = os.path.join(os.path.dirname(abi.library_path()), "librocmkernels_cache_gpu_check.so")
    if not os.path.exists(path):
        pytest.fail(f"{path} is missing: build it with __graft_entry__.build() (CMake)")
    abi.lib()
    S, P, I = abi.Strides, ctypes.c_void_p, ctypes.c_int
    step = ctypes.CDLL(path).cache_step
    step.argtypes = [P] * 8 + [abi.Cache, abi.Sequences, I, I, I, I, I] + [S] * 6 + [ctypes.c_ubyte, P, ctypes.c_ulonglong, P]
    step.restype = ctypes.c_longlong
    heads, width, size, tokens = 2, 64, 32, 45
    table, starts, ends = batch_of(device, [1, 44], [3000, 50], size, 120, 3)
    flat = noise(1, tokens, 8, width).to(torch.bfloat16).to(device)  # q, k and v in one tensor: strides that differ from packed ones
    q, k, v = flat[:, :4], flat[:, 4:6], flat[:, 6:]
    cos, sin = (t.to(device) for t in tables(3000, width + 8))
    cos = cos[:, :width]
    sin = sin.contiguous()[:, 4:4 + width]
    caches = [filled_cache(device, 120, size, heads, width, 5) for _ in range(2)]
    want_q = kv.append(caches[0], k, v, table, starts, ends, q=q, cos=cos, sin=sin)
    want, want_lse = kv.attention(caches[0], want_q, table, starts, ends, radius=2500)
    out_q, output, lse = torch.empty_like(want_q), torch.empty_like(want), torch.empty_like(want_lse)
    workspace = kv.workspace(caches[1], q, table)
    s = lambda t: S(0, t.stride(1) if t.dim() == 3 else 0, t.stride(0))  # noqa: E731
    sequences = abi.Sequences(starts.data_ptr(), ends.data_ptr(), table.data_ptr(), 2, tokens, table.shape[1], table.stride(0))
    need = step(k.data_ptr(), v.data_ptr(), q.data_ptr(), cos.data_ptr(), sin.data_ptr(), out_q.data_ptr(), output.data_ptr(), lse.data_ptr(),
                caches[1]._struct, sequences, 4, 3000, 0, 2500, 1, s(k), s(v), s(q), s(out_q), s(cos), s(sin), abi.DTYPE_BFLOAT16,
                workspace.data_ptr(), workspace.numel(), torch.cuda.current_stream().cuda_stream)
    assert need == workspace.numel() > 0
    torch.cuda.synchronize()
    assert torch.equal(out_q, want_q) and torch.equal(output, want) and torch.equal(lse, want_lse)
    for name in ("keys", "values"):
        assert torch.equal(getattr(caches[0], name).view(torch.uint8), getattr(caches[1], name).view(torch.uint8))
    assert torch.equal(caches[0].scales, caches[1].scales)


def test_no_rows(device):
    cache = filled_cache(device, 4, 16, 2, 32, 62)
    before = cache.keys.view(torch.uint8).clone()
    table, ends = torch.zeros((2, 3), dtype=torch.int32, device=device), torch.tensor([4, 5], dtype=torch.int32, device=device)
    starts = torch.zeros(3, dtype=torch.int32, device=device)
    none = torch.empty((0, 2, 32), device=device)
    assert kv.append(cache, none, none, table, starts, ends) is None
    output, lse = kv.attention(cache, none, table, starts, ends)
    assert output.shape == (0, 2, 32) and lse.shape == (0, 2, 2)
    some = torch.full((3, 2, 32), 5.0, device=device)  # rows, but of no sequence
    kv.append(cache, some, some, table, starts, ends)
    output, _ = kv.attention(cache, some, table, starts, ends, output=some.clone())
    torch.cuda.synchronize()
    assert torch.equal(cache.keys.view(torch.uint8), before) and (output == 5.0).all()


# ---- refusals -----------------------------------------------------------------------------------------------------
def test_refusals(device):
    cache = filled_cache(device, 4, 32, 2, 64, 63)
    table, starts, ends = batch_of(device, [2, 1], [20, 9], 32, 4, 1)
    k, q = torch.zeros((3, 2, 64), device=device), torch.zeros((3, 4, 64), device=device)
    cos = torch.zeros((64, 64), device=device)
    good = dict(q=q, cos=cos, sin=cos)
    bad_appends = [
        (k.half(), k, table, starts, ends, good), (k.double(), k.double(), table, starts, ends, {}), (k[:, :1], k[:, :1], table, starts, ends, {}),
        (k, k[:2], table, starts, ends, {}), (k, k, table.long(), starts, ends, {}), (k, k, table, starts[:-1], ends, {}),
        (k, k, table, starts, ends[:1], {}), (k, k, table, starts, ends, dict(q=q)), (k, k, table, starts, ends, dict(cos=cos)),
        (k, k, table, starts, ends, dict(good, cos=cos[:, :32])), (k, k, table, starts, ends, dict(good, sin=cos[:9])),
        (k, k, table, starts, ends, dict(good, q=q.half())), (k, k, table, starts, ends, dict(out_q=q)),
        (k.cpu(), k, table, starts, ends, {}), (k, k, table.cpu(), starts, ends, {}), (k, k, table, starts, ends.cpu(), {}),
        (k.transpose(1, 2).contiguous().transpose(1, 2), k, table, starts, ends, {}), (k, k, table.T, starts, ends, {}),
        (k, k, table, starts, ends, dict(good, q=q.cpu())), (k, k, table, starts, ends, dict(good, cos=cos.half())),
    ]
    for n, (a, b, t, s, e, more) in enumerate(bad_appends):
        with pytest.raises(ValueError):
            kv.append(cache, a, b, t, s, e, **more)
            pytest.fail(f"append {n} was accepted")
    odd = torch.zeros((3, 3, 64), device=device)
    for n, (x, more) in enumerate([(odd, {}), (q[..., :32], {}), (q[0], {}), (q.double(), {}), (q, dict(output=q.half())),
                                   (q, dict(lse=torch.zeros((3, 4), device=device))), (q, dict(output=q[:2])), (q.cpu(), {}),
                                   (q, dict(workspace=torch.zeros(8, dtype=torch.uint8))), (q[:, :0], {})]):
        with pytest.raises(ValueError):
            kv.attention(cache, x, table, starts, ends, **more)
            pytest.fail(f"attention {n} was accepted")
    for more in (dict(radius=-2), dict(max_keys=-1)):
        with pytest.raises(abi.HipError):
            kv.attention(cache, q, table, starts, ends, **more)
    long_table = torch.zeros((1, 500), dtype=torch.int32, device=device)
    need = kv.workspace(cache, q[:1], long_table)
    assert need.numel() > 0
    with pytest.raises(abi.HipError):
        kv.attention(cache, q[:1], long_table, starts[:2], ends[:1], workspace=need[:need.numel() // 8])
    for wrong in (dict(width=48), dict(page_size=24), dict(page_size=144), dict(heads=0)):
        with pytest.raises(ValueError):
            kv.KVCache.empty(**dict(dict(pages=2, page_size=32, heads=2, width=64, device=device), **wrong))
    keys, values, scales = cache.keys, cache.values, cache.scales
    for a, b, c in ((keys.view(torch.uint8), values, scales), (keys[:3], values, scales), (keys, keys, scales), (keys, values, scales[:, :1]),
                    (keys, values, scales.half()), (keys.cpu(), values.cpu(), scales.cpu()), (keys[:, :1], values[:, :1], scales[:, :1])):
        with pytest.raises(ValueError):
            kv.KVCache(a, b, c)
