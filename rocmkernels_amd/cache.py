"""Paged 8-bit key/value cache: appending tokens with the position rotation applied on the way, and attention over the cache.

For a model that answers: ``append`` quantises the new keys and values of a batch of sequences into their pages (rotating K, and
Q beside it), ``attention`` lets the new rows attend to everything their sequence holds. Both take the same description of the
batch, so one scheduler state serves a step:

* rows are packed: q [tokens][query heads][D], k and v [tokens][heads][D], float32, float16 or bfloat16, strided views with
  contiguous features; sequence b owns rows ``starts[b]`` .. ``starts[b + 1]`` - 1 (``starts`` int32 [batch + 1]);
* ``lengths[b]`` (int32 [batch]) counts the keys of sequence b with these rows, so row i of its n stands at position
  lengths[b] - n + i;
* ``table[b][p]`` (int32 [batch][columns]) is the page that holds positions p * page_size .. (p + 1) * page_size - 1.

A page keeps, for every K/V head, e4m3 keys and values with a power-of-two scale each (include/rocmkernels_cache.h has the layout
and the exact rules). Single tokens, drafted tokens, prompts, chunks of prompts and batches that mix them go through the same two
calls. Everything runs on the GPU through the C ABI, on the current stream of the tensors' device unless ``stream`` is given;
there is no CPU path. Nothing is copied to the host: what starts, lengths and table hold is not checked here (the kernels
keep to the buffers whatever they hold).
"""
import ctypes
import functools

from . import attention as _abi

_DTYPES = {}  # torch dtype -> rocmkernels_dtype, filled on first use


def _dtype(t, name):
    if not _DTYPES:
        torch = _abi._torch()
        _DTYPES.update({torch.float32: _abi.DTYPE_FLOAT32, torch.float16: _abi.DTYPE_FLOAT16, torch.bfloat16: _abi.DTYPE_BFLOAT16})
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}") from None


@functools.lru_cache(maxsize=512)
def _shared_strides(head, token):
    if not (-(1 << 31) <= head < 1 << 31 and -(1 << 31) <= token < 1 << 31):
        raise ValueError("strides must fit 32 bits")
    return _abi.Strides(0, head, token)


def _rows(t, name, heads, width, tokens=None, like=None):
    """Strides of a [tokens][heads][width] view with contiguous features, checked against what it has to agree with."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != width or shape[1] != heads or (tokens is not None and shape[0] != tokens):
        raise ValueError(f"{name} must be [{'tokens' if tokens is None else tokens}][{heads}][{width}], not {tuple(shape)}")
    if like is not None and t.dtype != like.dtype:
        raise ValueError(f"{name} must be {like.dtype}, not {t.dtype}")
    s = t.stride()
    if s[2] != 1:
        raise ValueError(f"{name} must have contiguous features")
    return _shared_strides(s[1], s[0])


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.get_device() != device:
            raise ValueError(f"{name} must be on the cache's device (cuda:{device})")


class KVCache:
    """The tensors of a paged cache: ``keys`` float8_e4m3fn [page][head][P / 16][16][D], ``values`` float8_e4m3fn
    [page][head][P / 16][D][16] (16-token blocks transposed) and ``scales`` float32 [page][head][2]; P tokens to a page."""

    def __init__(self, keys, values, scales):
        torch = _abi._torch()
        if keys.dtype != torch.float8_e4m3fn or values.dtype != torch.float8_e4m3fn or scales.dtype != torch.float32:
            raise ValueError("keys and values must be float8_e4m3fn and scales float32")
        if keys.dim() != 5 or keys.shape[3] != 16:
            raise ValueError(f"keys must be [page][head][blocks][16][width], not {tuple(keys.shape)}")
        pages, heads, blocks, _, width = keys.shape
        if width not in (32, 64, 128) or not 1 <= blocks <= 8 or pages < 1 or heads < 1:
            raise ValueError("a cache has at least one page and head, 16 to 128 tokens to a page, and width 32, 64 or 128")
        if values.shape != (pages, heads, blocks, width, 16) or scales.shape != (pages, heads, 2):
            raise ValueError(f"values must be {(pages, heads, blocks, width, 16)} and scales {(pages, heads, 2)}")
        if not (keys.is_contiguous() and values.is_contiguous() and scales.is_contiguous()):
            raise ValueError("the cache's tensors must be contiguous")
        if not keys.is_cuda:
            raise ValueError("the cache kernels run on the GPU only; move the tensors to a HIP device")
        if keys.data_ptr() % 16 or values.data_ptr() % 16 or scales.data_ptr() % 8:
            raise ValueError("keys and values must be 16-byte aligned, scales 8-byte")
        self._device = keys.get_device()
        _same_device(self._device, values=values, scales=scales)
        self.keys, self.values, self.scales = keys, values, scales
        self.pages, self.heads, self.page_size, self.width = pages, heads, 16 * blocks, width
        self._struct = _abi.Cache(keys.data_ptr(), values.data_ptr(), scales.data_ptr(), pages, 16 * blocks, heads, width)

    @classmethod
    def empty(cls, pages, page_size, heads, width, device="cuda"):
        """A cache of its own with no tokens in it."""
        torch = _abi._torch()
        if page_size % 16 or not 16 <= page_size <= 128:
            raise ValueError("page_size must be a multiple of 16 from 16 to 128")
        blocks = page_size // 16
        keys = torch.zeros((pages, heads, blocks, 16, width), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        values = torch.zeros((pages, heads, blocks, width, 16), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        return cls(keys, values, torch.zeros((pages, heads, 2), dtype=torch.float32, device=device))


def _sequences(cache, table, starts, lengths, tokens):
    torch = _abi._torch()
    int32 = torch.int32
    if table.dtype != int32 or starts.dtype != int32 or lengths.dtype != int32:
        raise ValueError("table, starts and lengths must be int32")
    shape = table.shape
    if len(shape) != 2 or starts.shape != (shape[0] + 1,) or lengths.shape != (shape[0],):
        raise ValueError("table must be [batch][columns], starts [batch + 1] and lengths [batch]")
    s = table.stride()
    if (s[1] != 1 and shape[1] > 1) or (s[0] < shape[1] and shape[0] > 1):
        raise ValueError("table must have contiguous rows")
    if not starts.is_contiguous() or not lengths.is_contiguous():
        raise ValueError("starts and lengths must be contiguous")
    device = cache._device
    if table.get_device() != device or starts.get_device() != device or lengths.get_device() != device:
        _same_device(device, table=table, starts=starts, lengths=lengths)
    return _abi.Sequences(starts.data_ptr(), lengths.data_ptr(), table.data_ptr(), shape[0], tokens, shape[1], max(s[0], shape[1]))


def _on(cache, stream, work):
    """Calls work(stream handle) with the cache's device current, and ``stream`` for what it allocates."""
    torch = _abi._torch()
    if stream is None and torch._C._cuda_getDevice() == cache._device:
        return work(torch._C._cuda_getCurrentRawStream(cache._device))
    if stream is None:
        with torch.cuda.device(cache._device):
            return work(torch._C._cuda_getCurrentRawStream(cache._device))
    if stream.device.index != cache._device:
        raise ValueError(f"stream must belong to the cache's device (cuda:{cache._device})")
    with torch.cuda.stream(stream):  # switches the device too
        return work(stream.cuda_stream)


def _table(t, name, width):
    torch = _abi._torch()
    shape, s = t.shape, t.stride()
    if t.dtype != torch.float32 or len(shape) != 2 or shape[1] != width or s[1] != 1:
        raise ValueError(f"{name} must be a float32 [positions][{width}] table with contiguous columns")
    return _shared_strides(0, s[0])


def append(cache, k, v, table, starts, lengths, q=None, cos=None, sin=None, out_q=None, stream=None):
    """Appends k and v [tokens][heads][D] to ``cache`` and returns the rotated queries (None without ``q``).

    With ``cos`` and ``sin`` (float32 [positions][D], rows by position, in rotary's convention) K is rotated before it is
    quantised; with ``q`` [tokens][query heads][D] the queries are rotated too, into ``out_q`` (which may be ``q``; allocated
    when None). A page's scale is the smallest power of two that holds its new values, or the scale the page had, if larger; earlier
    rows are requantised when it grows. Rows outside every sequence, at a position past the table's columns or past cos and sin
    are left out (their rows of ``out_q`` are left as they were)."""
    torch = _abi._torch()
    dtype, tokens = _dtype(k, "k"), k.shape[0]
    ks = _rows(k, "k", cache.heads, cache.width)
    vs = _rows(v, "v", cache.heads, cache.width, tokens, k)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if q is not None and cos is None:
        raise ValueError("queries are rotated: q needs cos and sin")
    if q is None and out_q is not None:
        raise ValueError("out_q needs q")
    none = _shared_strides(0, 0)
    cs = ss = qs = none
    positions = query_heads = 0
    if cos is not None:
        cs, ss, positions = _table(cos, "cos", cache.width), _table(sin, "sin", cache.width), cos.shape[0]
        if sin.shape != cos.shape:
            raise ValueError("cos and sin must have the same shape")
    if q is not None:
        query_heads = q.shape[1] if q.dim() == 3 else 0
        qs = _rows(q, "q", query_heads, cache.width, tokens, k)
        if out_q is not None:
            _rows(out_q, "out_q", query_heads, cache.width, tokens, k)
    _same_device(cache._device, k=k, v=v, q=q, cos=cos, sin=sin, out_q=out_q)
    sequences = _sequences(cache, table, starts, lengths, tokens)

    def work(handle):
        out = torch.empty((tokens, query_heads, cache.width), dtype=q.dtype, device=q.device) if q is not None and out_q is None else out_q
        os = none if out is None else _rows(out, "out_q", query_heads, cache.width)
        if tokens:
            _abi.check("attention_cache_append", k.data_ptr(), v.data_ptr(), _abi._ptr(q), _abi._ptr(cos), _abi._ptr(sin), _abi._ptr(out),
                       cache._struct, sequences, query_heads, positions, ks, vs, qs, os, cs, ss, dtype, handle)
        return out

    return _on(cache, stream, work)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(page_size, heads, width, batch, tokens, columns, query_heads, max_keys, dtype):
    size = ctypes.c_size_t()
    _abi.check("attention_cache_workspace", _abi.Cache(None, None, None, 1, page_size, heads, width),
               _abi.Sequences(None, None, None, batch, tokens, columns, columns), query_heads, max_keys, dtype, ctypes.byref(size))
    return size.value


def workspace(cache, q, table, max_keys=0):
    """A workspace for ``attention`` on tensors of these shapes, any window: a uint8 tensor, empty where none is needed. Calls that may
    run at the same time need one each."""
    torch = _abi._torch()
    size = _workspace_bytes(cache.page_size, cache.heads, cache.width, table.shape[0], q.shape[0], table.shape[1], q.shape[1],
                            int(max_keys), _dtype(q, "q"))
    return torch.empty(size, dtype=torch.uint8, device=cache.keys.device)


def attention(cache, q, table, starts, lengths, causal=True, radius=-1, max_keys=0, output=None, lse=None, workspace=None,
              stream=None):
    """output, lse of the query rows q [tokens][query heads][D] over the keys their sequences hold in ``cache``.

    Query head i reads K/V head i / (query heads / heads). ``causal`` lets a row see keys up to its own position, ``radius`` >= 0
    keys within that distance. ``max_keys`` is a bound on the keys of every sequence that the caller knows (0: what the table can
    hold); it shapes the launch, and keys behind it are not seen. output has q's type, lse is float32 [tokens][query
    heads][2] = {maximum of the scaled scores, sum of exp(score - maximum)}; a row that sees no key gets 0 and {-inf, 0}; rows outside
    every sequence are left as they were. ``workspace`` (see ``workspace``) is allocated when None."""
    torch = _abi._torch()
    if q.dim() != 3:
        raise ValueError(f"q must be [tokens][query heads][{cache.width}], not {tuple(q.shape)}")
    dtype, (tokens, query_heads, _) = _dtype(q, "q"), q.shape
    qs = _rows(q, "q", query_heads, cache.width)
    if query_heads == 0 or query_heads % cache.heads:
        raise ValueError(f"{query_heads} query heads do not share {cache.heads} K/V heads evenly")
    if output is not None:
        _rows(output, "output", query_heads, cache.width, tokens, q)
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (tokens, query_heads, 2) or not lse.is_contiguous()):
        raise ValueError(f"lse must be a contiguous float32 [{tokens}][{query_heads}][2] tensor")
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    _same_device(cache._device, q=q, output=output, lse=lse, workspace=workspace)
    sequences = _sequences(cache, table, starts, lengths, tokens)
    columns = table.shape[1]

    def work(handle):
        out = torch.empty((tokens, query_heads, cache.width), dtype=q.dtype, device=q.device) if output is None else output
        statistics = torch.empty((tokens, query_heads, 2), dtype=torch.float32, device=q.device) if lse is None else lse
        scratch = workspace
        if scratch is None and tokens:
            size = _workspace_bytes(cache.page_size, cache.heads, cache.width, table.shape[0], tokens, columns, query_heads,
                                    int(max_keys), dtype)
            scratch = torch.empty(size, dtype=torch.uint8, device=q.device)
        if tokens:
            _abi.check("attention_cache_forward", q.data_ptr(), cache._struct, sequences, out.data_ptr(), statistics.data_ptr(), query_heads,
                       int(max_keys), int(radius), _abi.CAUSAL if causal else 0, qs, _rows(out, "output", query_heads, cache.width), dtype,
                       scratch.data_ptr(), scratch.numel() * scratch.element_size(), handle)
        return out, statistics

    return _on(cache, stream, work)
