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

_torch = _abi._torch  # the module, imported on first use
_NONE = _abi.Strides(0, 0, 0)


@functools.lru_cache(maxsize=None)
def _constants():
    """(torch dtype -> rocmkernels_dtype, int32, float32, the current device's index, a device's current stream, the library)."""
    torch, lib = _torch(), _abi.lib()
    codes = {torch.float32: _abi.DTYPE_FLOAT32, torch.float16: _abi.DTYPE_FLOAT16, torch.bfloat16: _abi.DTYPE_BFLOAT16}
    return codes, torch.int32, torch.float32, torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream, lib


@functools.lru_cache(maxsize=512)
def _strides(strides):
    """The struct for strides (token, head, 1) or (row, 1), shared between equal ones."""
    if strides[-1] != 1:
        raise ValueError("features must be contiguous")
    head = strides[1] if len(strides) == 3 else 0
    if not (-(1 << 31) <= head < 1 << 31 and -(1 << 31) <= strides[0] < 1 << 31):
        raise ValueError("strides must fit 32 bits")
    return _abi.Strides(0, head, strides[0])


# A small call is bound by what is done here, so the calls below check in straight lines and name what is wrong only once something
# is: host time without the launch, of an append with queries 9.8 µs where a helper for each check took 14.9, of an attention
# call 7.2 (10.9).
def _wrong_rows(name, t, shape, dtype):
    raise ValueError(f"{name} must be {list(shape)} of {dtype}, not {list(t.shape)} of {t.dtype}")


def _wrong_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.get_device() != device:
            raise ValueError(f"{name} must be on the cache's device (cuda:{device})")


def _wrong_sequences(table, starts, lengths):
    int32 = _torch().int32
    if table.dtype != int32 or starts.dtype != int32 or lengths.dtype != int32:
        raise ValueError("table, starts and lengths must be int32")
    shape, s = table.shape, table.stride()
    if len(shape) != 2 or starts.shape != (shape[0] + 1,) or lengths.shape != (shape[0],):
        raise ValueError("table must be [batch][columns], starts [batch + 1] and lengths [batch]")
    if s[1] != 1 or s[0] < shape[1]:
        raise ValueError("table must have contiguous rows that do not overlap")
    raise ValueError("starts and lengths must be contiguous")


def _elsewhere(cache, stream, call, *args, **more):
    """The call on ``stream``, or on the current stream of a device that is not the current one."""
    torch = _torch()
    if stream is None:
        with torch.cuda.device(cache._device):
            return call(cache, *args, **more)
    if stream.device.index != cache._device:
        raise ValueError(f"stream must belong to the cache's device (cuda:{cache._device})")
    with torch.cuda.stream(stream):  # what the call allocates belongs to the stream too
        return call(cache, *args, **more)


class KVCache:
    """The tensors of a paged cache: ``keys`` float8_e4m3fn [page][head][P / 16][16][D], ``values`` float8_e4m3fn
    [page][head][P / 16][D][16] (16-token blocks transposed) and ``scales`` float32 [page][head][2]; P tokens to a page."""

    def __init__(self, keys, values, scales):
        torch = _torch()
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
        _wrong_device(self._device, values=values, scales=scales)
        self.keys, self.values, self.scales = keys, values, scales
        self.pages, self.heads, self.page_size, self.width = pages, heads, 16 * blocks, width
        self._struct = _abi.Cache(keys.data_ptr(), values.data_ptr(), scales.data_ptr(), pages, 16 * blocks, heads, width)

    @classmethod
    def empty(cls, pages, page_size, heads, width, device="cuda"):
        """A cache of its own with no tokens in it."""
        torch = _torch()
        if page_size % 16 or not 16 <= page_size <= 128:
            raise ValueError("page_size must be a multiple of 16 from 16 to 128")
        blocks = page_size // 16
        keys = torch.zeros((pages, heads, blocks, 16, width), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        values = torch.zeros((pages, heads, blocks, width, 16), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        return cls(keys, values, torch.zeros((pages, heads, 2), dtype=torch.float32, device=device))


def _sequences(table, starts, lengths, tokens, int32):
    shape, strides = table.shape, table.stride()
    batch = shape[0]
    if (len(shape) != 2 or table.dtype != int32 or starts.dtype != int32 or lengths.dtype != int32 or starts.shape != (batch + 1,)
            or lengths.shape != (batch,) or strides[1] != 1 or strides[0] < shape[1] or not starts.is_contiguous()
            or not lengths.is_contiguous()):
        _wrong_sequences(table, starts, lengths)
    return _abi.Sequences(starts.data_ptr(), lengths.data_ptr(), table.data_ptr(), batch, tokens, shape[1], strides[0])


def append(cache, k, v, table, starts, lengths, q=None, cos=None, sin=None, out_q=None, stream=None):
    """Appends k and v [tokens][heads][D] to ``cache`` and returns the rotated queries (None without ``q``).

    With ``cos`` and ``sin`` (float32 [positions][D], rows by position, in rotary's convention) K is rotated before it is
    quantised; with ``q`` [tokens][query heads][D] the queries are rotated too, into ``out_q`` (which may be ``q``; allocated
    when None). A page's scale is the smallest power of two that holds its new values, or the scale the page had, if larger; earlier
    rows are requantised when it grows. Rows outside every sequence, at a position past the table's columns or past cos and sin
    are left out (their rows of ``out_q`` are left as they were)."""
    codes, int32, float32, current_device, current_stream, lib = _constants()
    device = cache._device
    if stream is not None or current_device() != device:
        return _elsewhere(cache, stream, append, k, v, table, starts, lengths, q=q, cos=cos, sin=sin, out_q=out_q)
    width, shape, dtype = cache.width, k.shape, k.dtype
    tokens, code = shape[0], codes.get(dtype)
    if code is None:
        raise ValueError(f"k must be float32, float16 or bfloat16, not {dtype}")
    if len(shape) != 3 or shape[1] != cache.heads or shape[2] != width:
        _wrong_rows("k", k, ("tokens", cache.heads, width), dtype)
    if v.shape != shape or v.dtype != dtype:
        _wrong_rows("v", v, shape, dtype)
    if (k.get_device() != device or v.get_device() != device or table.get_device() != device or starts.get_device() != device
            or lengths.get_device() != device):
        _wrong_device(device, k=k, v=v, table=table, starts=starts, lengths=lengths)
    sequences = _sequences(table, starts, lengths, tokens, int32)
    cs = ss = qs = os = _NONE
    cos_at = sin_at = q_at = out_at = None
    positions = query_heads = 0
    if cos is not None or sin is not None:
        if cos is None or sin is None:
            raise ValueError("cos and sin come together")
        span = cos.shape
        if len(span) != 2 or span[1] != width or sin.shape != span or cos.dtype != float32 or sin.dtype != float32:
            raise ValueError(f"cos and sin must be float32 [positions][{width}] tables of one shape")
        if cos.get_device() != device or sin.get_device() != device:
            _wrong_device(device, cos=cos, sin=sin)
        positions, cs, ss, cos_at, sin_at = span[0], _strides(cos.stride()), _strides(sin.stride()), cos.data_ptr(), sin.data_ptr()
    if q is None:
        if out_q is not None:
            raise ValueError("out_q needs q")
    else:
        if cos is None:
            raise ValueError("queries are rotated: q needs cos and sin")
        shape = q.shape
        if len(shape) != 3 or shape[0] != tokens or shape[2] != width or q.dtype != dtype:
            _wrong_rows("q", q, (tokens, "query heads", width), dtype)
        query_heads = shape[1]
        if query_heads == 0 or query_heads % cache.heads:
            raise ValueError(f"{query_heads} query heads do not share {cache.heads} K/V heads evenly")
        if out_q is None:
            out_q = _torch().empty(shape, dtype=dtype, device=q.device)
        elif out_q.shape != shape or out_q.dtype != dtype:
            _wrong_rows("out_q", out_q, shape, dtype)
        if q.get_device() != device or out_q.get_device() != device:
            _wrong_device(device, q=q, out_q=out_q)
        qs, os, q_at, out_at = _strides(q.stride()), _strides(out_q.stride()), q.data_ptr(), out_q.data_ptr()
    if tokens:
        status = lib.attention_cache_append(k.data_ptr(), v.data_ptr(), q_at, cos_at, sin_at, out_at, cache._struct, sequences, query_heads,
                                            positions, _strides(k.stride()), _strides(v.stride()), qs, os, cs, ss, code, current_stream(device))
        if status:
            raise _abi.HipError(status, "attention_cache_append")
    return out_q


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(page_size, heads, width, batch, tokens, columns, query_heads, max_keys, dtype):
    size = ctypes.c_size_t()
    _abi.check("attention_cache_workspace", _abi.Cache(None, None, None, 1, page_size, heads, width),
               _abi.Sequences(None, None, None, batch, tokens, columns, columns), query_heads, max_keys, dtype, ctypes.byref(size))
    return size.value


def workspace(cache, q, table, max_keys=0):
    """A workspace for ``attention`` on tensors of these shapes, any window: a uint8 tensor, empty where none is needed. Calls that may
    run at the same time need one each."""
    torch = _torch()
    if len(q.shape) != 3 or q.dtype not in _constants()[0] or len(table.shape) != 2:
        raise ValueError("q must be [tokens][query heads][width] of float32, float16 or bfloat16, and table [batch][columns]")
    size = _workspace_bytes(cache.page_size, cache.heads, cache.width, table.shape[0], q.shape[0], table.shape[1], q.shape[1],
                            int(max_keys), _constants()[0][q.dtype])
    return torch.empty(size, dtype=torch.uint8, device=cache.keys.device)


def attention(cache, q, table, starts, lengths, causal=True, radius=-1, max_keys=0, output=None, lse=None, workspace=None,
              stream=None):
    """output, lse of the query rows q [tokens][query heads][D] over the keys their sequences hold in ``cache``.

    Query head i reads K/V head i / (query heads / heads). ``causal`` lets a row see keys up to its own position, ``radius`` >= 0
    keys within that distance. ``max_keys`` is a bound on the keys of every sequence that the caller knows (0: what the table can
    hold); it shapes the launch, and keys behind it are not seen. output has q's type, lse is float32 [tokens][query
    heads][2] = {maximum of the scaled scores, sum of exp(score - maximum)}; a row that sees no key gets 0 and {-inf, 0}; rows outside
    every sequence are left as they were. ``workspace`` (see ``workspace``) is allocated when None."""
    codes, int32, float32, current_device, current_stream, lib = _constants()
    device = cache._device
    if stream is not None or current_device() != device:
        return _elsewhere(cache, stream, attention, q, table, starts, lengths, causal=causal, radius=radius, max_keys=max_keys, output=output,
                          lse=lse, workspace=workspace)
    width, shape, dtype = cache.width, q.shape, q.dtype
    code = codes.get(dtype)
    if code is None:
        raise ValueError(f"q must be float32, float16 or bfloat16, not {dtype}")
    if len(shape) != 3 or shape[2] != width:
        _wrong_rows("q", q, ("tokens", "query heads", width), dtype)
    tokens, query_heads = shape[0], shape[1]
    if query_heads == 0 or query_heads % cache.heads:
        raise ValueError(f"{query_heads} query heads do not share {cache.heads} K/V heads evenly")
    if (q.get_device() != device or table.get_device() != device or starts.get_device() != device or lengths.get_device() != device):
        _wrong_device(device, q=q, table=table, starts=starts, lengths=lengths)
    sequences = _sequences(table, starts, lengths, tokens, int32)
    if output is None:
        output = _torch().empty(shape, dtype=dtype, device=q.device)
    elif output.shape != shape or output.dtype != dtype:
        _wrong_rows("output", output, shape, dtype)
    if lse is None:
        lse = _torch().empty((tokens, query_heads, 2), dtype=float32, device=q.device)
    elif lse.shape != (tokens, query_heads, 2) or lse.dtype != float32 or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 [{tokens}][{query_heads}][2] tensor")
    if workspace is None:
        size = _workspace_bytes(cache.page_size, cache.heads, width, sequences.batch, tokens, sequences.columns, query_heads, int(max_keys), code)
        workspace = _torch().empty(size, dtype=_torch().uint8, device=q.device)
    elif not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    if output.get_device() != device or lse.get_device() != device or workspace.get_device() != device:
        _wrong_device(device, output=output, lse=lse, workspace=workspace)
    if tokens:
        status = lib.attention_cache_forward(q.data_ptr(), cache._struct, sequences, output.data_ptr(), lse.data_ptr(), query_heads,
                                             max_keys, radius, _abi.CAUSAL if causal else 0, _strides(q.stride()), _strides(output.stride()),
                                             code, workspace.data_ptr(), workspace.nbytes, current_stream(device))
        if status:
            raise _abi.HipError(status, "attention_cache_forward")
    return output, lse
