"""The 8-bit KV cache over torch CUDA tensors: quantising append, attention over
it, block selection and sparse attention (n550_kv8_*, n550_attention_*_kv8)."""
from __future__ import annotations

import ctypes as C

from . import BF16, F32, KV8_BLOCK, KV8CacheStruct, check, lib

_LAYERS, _NKV, _HD, _NH = 28, 8, 128, 16


def _stream(cache, *tensors):
    """The raw current stream of the cache's device, which must be the current one
    and hold the tensors."""
    import torch
    dev = cache.device_index
    for t in tensors:
        if t.get_device() != dev:
            raise ValueError(f"tensor on {t.device}, but the cache is on cuda:{dev}")
    if torch.cuda.current_device() != dev:
        raise ValueError(f"the cache is on cuda:{dev}, the current device is cuda:{torch.cuda.current_device()}")
    return torch._C._cuda_getCurrentRawStream(dev)


class KV8Cache:
    """K and V of n_slots sequences as e4m3 codes with a scale per block of 64
    positions and KV head (n550_kv8_cache). Tensors: k, v [n_slots, n_layers, 8,
    max_len, 128] float8_e4m3fn, k_scale, v_scale [n_slots, n_layers, 8, n_blocks]
    float32, k_bounds [n_slots, n_layers, 8, n_blocks, 2, 128] float8_e4m3fn or
    None. Allocated here, or handed over by keyword; the calls below read and write
    these tensors' memory, so another tensor cannot take one's place."""

    k, v = property(lambda c: c._tensors[0]), property(lambda c: c._tensors[1])
    k_scale, v_scale = property(lambda c: c._tensors[2]), property(lambda c: c._tensors[3])
    k_bounds = property(lambda c: c._tensors[4])

    def __init__(self, n_slots=None, max_len=None, n_layers=_LAYERS, device="cuda", bounds=True, *,
                 k=None, v=None, k_scale=None, v_scale=None, k_bounds=None):
        import torch
        e4 = torch.float8_e4m3fn
        given = [k, v, k_scale, v_scale]
        if all(t is None for t in given) and k_bounds is None:
            if n_slots is None or max_len is None or min(n_slots, max_len, n_layers) < 1:
                raise ValueError("n_slots, max_len and n_layers must be at least 1")
            nb = -(-max_len // KV8_BLOCK)
            plane = (n_slots, n_layers, _NKV)
            k = torch.empty(plane + (max_len, _HD), dtype=e4, device=device)
            v = torch.empty_like(k)
            k_scale = torch.empty(plane + (nb,), dtype=torch.float32, device=device)
            v_scale = torch.empty_like(k_scale)
            if bounds:
                k_bounds = torch.empty(plane + (nb, 2, _HD), dtype=e4, device=device)
        elif any(t is None for t in given):
            raise ValueError("k, v, k_scale and v_scale belong together")
        if k.dim() != 5 or k.shape[2] != _NKV or k.shape[4] != _HD:
            raise ValueError("KV cache must be [slots, layers, 8, max_len, 128]")
        nb = -(-k.shape[3] // KV8_BLOCK)
        plane = tuple(k.shape[:3])
        want = {"k": (k, tuple(k.shape), e4), "v": (v, tuple(k.shape), e4),
                "k_scale": (k_scale, plane + (nb,), torch.float32),
                "v_scale": (v_scale, plane + (nb,), torch.float32),
                "k_bounds": (k_bounds, plane + (nb, 2, _HD), e4)}
        for name, (t, shape, dt) in want.items():
            if t is None and name == "k_bounds":
                continue
            if tuple(t.shape) != shape or t.dtype != dt or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dt} tensor of shape {shape}")
            if t.device.type != "cuda" or t.device != k.device:
                raise ValueError("the cache's tensors must be on one CUDA device")
        self._tensors = (k, v, k_scale, v_scale, k_bounds)
        self.n_slots, self.n_layers, self.max_len, self.n_blocks = k.shape[0], k.shape[1], k.shape[3], nb
        self.device_index = k.get_device()
        self._c = KV8CacheStruct(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                 k_bounds.data_ptr() if k_bounds is not None else None,
                                 self.n_slots, self.n_layers, self.max_len)
        self._ref = C.byref(self._c)


def _ids(seq_ids, pos=None):
    """Number of sequences; both must be contiguous int32 vectors of that length."""
    import torch
    i32 = torch.int32
    if seq_ids.dim() != 1 or seq_ids.dtype != i32 or not seq_ids.is_contiguous():
        raise ValueError("seq_ids must be a contiguous int32 vector")
    n = seq_ids.numel()
    if pos is not None and (pos.dim() != 1 or pos.numel() != n or pos.dtype != i32 or not pos.is_contiguous()):
        raise ValueError(f"pos must be a contiguous int32 vector of {n}")
    return n


_INT_MAX = 2 ** 31 - 1


def _c_int(name, x):
    """Numbers that the library takes as C ints: ctypes would cut larger ones to their
    lower 32 bits."""
    if not -_INT_MAX <= x <= _INT_MAX:
        raise ValueError(f"{name} = {x} does not fit 32 bits")


def _rows(name, t, rows, cols, dtypes):
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != rows or shape[1] < cols or t.dtype not in dtypes or \
            (stride[1] != 1 and rows > 0):
        raise ValueError(f"{name} must be [{rows}, >= {cols}] with contiguous rows of {dtypes}")
    if rows > 1 and stride[0] > _INT_MAX:
        raise ValueError(f"{name} must have a row stride below 2^31 elements")
    # the stride of a single row is never used; torch reports any number there
    return stride[0] if rows > 1 else cols


def kv8_append(cache, k, v, seq_ids, pos, L, layer):
    """Quantise len(seq_ids) x L rows of k and v ([n_seqs*L, >= 1024] float32 or
    bfloat16) into positions pos[s] .. pos[s]+L-1 of slot seq_ids[s]."""
    import torch
    _c_int("layer", layer)
    _c_int("L", L)
    st = _stream(cache, k, v, seq_ids, pos)
    n = _ids(seq_ids, pos)
    if L < 0:
        raise ValueError("L must not be negative")
    ld = _rows("k", k, n * L, _NKV * _HD, (torch.float32, torch.bfloat16))
    if _rows("v", v, n * L, _NKV * _HD, (k.dtype,)) != ld:
        raise ValueError("k and v must have the same row stride")
    check(lib().n550_kv8_append(st, cache._ref, layer, k.data_ptr(), v.data_ptr(),
                                F32 if k.dtype == torch.float32 else BF16, ld, seq_ids.data_ptr(),
                                pos.data_ptr(), n, L), "n550_kv8_append")


def _q_out(q, rows, out):
    import torch
    ldq = _rows("q", q, rows, _NH * _HD, (torch.bfloat16,))
    if out is None:
        w = _NH * _HD
        # (the cheaper call where q is such a matrix itself)
        return ldq, torch.empty_like(q) if ldq == w == q.shape[1] else q.new_empty((rows, w)), w
    return ldq, out, _rows("out", out, rows, _NH * _HD, (torch.bfloat16,))


def _workspace(nbytes, q):
    # in q's type: new_empty takes device and dtype over without parsing them
    return q.new_empty((nbytes + 1) // 2)


def attention_decode_kv8(q, cache, seq_ids, pos, layer, out=None, split=True):
    """One query per sequence (rows of q, BF16) at position pos[s] over the 8-bit
    cache; split=True passes a split-KV workspace, split=False runs one CTA per
    (sequence, KV head)."""
    n = _ids(seq_ids, pos)
    _c_int("layer", layer)
    ldq, out, ldo = _q_out(q, n, out)
    st = _stream(cache, q, seq_ids, pos, out)
    L = lib()
    nbytes = L.n550_attention_kv8_workspace(n) if split else 0
    ws = _workspace(nbytes, q) if nbytes else None
    check(L.n550_attention_decode_kv8(st, q.data_ptr(), ldq, cache._ref, layer, seq_ids.data_ptr(),
                                      pos.data_ptr(), n, out.data_ptr(), ldo, ws.data_ptr() if nbytes else None, nbytes),
          "n550_attention_decode_kv8")
    return out


def attention_sparse_kv8(q, cache, seq_ids, pos, blocks, layer, out=None, split=True):
    """attention_decode_kv8 over the positions <= pos[s] of the listed blocks only:
    blocks int32 [n_seqs, 8, n_select], entries outside the context skipped."""
    import torch
    n = _ids(seq_ids, pos)
    shape = blocks.shape
    if blocks.dtype != torch.int32 or len(shape) != 3 or shape[0] != n or shape[1] != _NKV or \
            not blocks.is_contiguous():
        raise ValueError(f"blocks must be a contiguous int32 tensor [{n}, 8, n_select]")
    _c_int("layer", layer)
    _c_int("n_select", shape[2])
    ldq, out, ldo = _q_out(q, n, out)
    st = _stream(cache, q, seq_ids, pos, blocks, out)
    L = lib()
    nbytes = L.n550_attention_kv8_workspace(n) if split else 0
    ws = _workspace(nbytes, q) if nbytes else None
    check(L.n550_attention_sparse_kv8(st, q.data_ptr(), ldq, cache._ref, layer, seq_ids.data_ptr(),
                                      pos.data_ptr(), blocks.data_ptr(), shape[2], n,
                                      out.data_ptr(), ldo, ws.data_ptr() if nbytes else None, nbytes), "n550_attention_sparse_kv8")
    return out


# Most bytes that attention_prefill_kv8 allocates as a workspace, if one sequence's
# context as BF16 (4096 bytes a position) is not more: above it, sequences in groups.
PREFILL_WORKSPACE_MAX = 4 << 30


def attention_prefill_kv8(q, cache, seq_ids, L, pos0, layer, out=None, workspace=True):
    """Causal attention of len(seq_ids) sequences x L queries (rows of q, BF16) at
    positions pos0.. over the 8-bit cache, which holds their K/V already."""
    n = _ids(seq_ids)
    _c_int("L", L)
    _c_int("pos0", pos0)
    _c_int("layer", layer)
    if L < 0:
        raise ValueError("L must not be negative")
    ldq, out, ldo = _q_out(q, n * L, out)
    st = _stream(cache, q, seq_ids, out)
    lb = lib()
    # (positions outside the cache need none: the call below refuses them)
    nbytes = lb.n550_attention_prefill_kv8_workspace(n, L, pos0) if workspace and pos0 + L <= cache.max_len else 0
    if nbytes > PREFILL_WORKSPACE_MAX:
        nbytes = min(nbytes, max(PREFILL_WORKSPACE_MAX, lb.n550_attention_prefill_kv8_workspace(1, L, pos0)))
    ws = _workspace(nbytes, q) if nbytes else None
    check(lb.n550_attention_prefill_kv8(st, q.data_ptr(), ldq, cache._ref, layer, seq_ids.data_ptr(), n,
                                        L, pos0, out.data_ptr(), ldo, ws.data_ptr() if nbytes else None, nbytes),
          "n550_attention_prefill_kv8")
    return out


def kv8_select_blocks(q, cache, seq_ids, pos, layer, n_select, n_sink=1, n_recent=2, out=None):
    """The n_select blocks of each context whose bounds promise the largest scores
    for the sequence's query, per KV head: int32 [n_seqs, 8, n_select], ascending,
    -1 behind the last."""
    import torch
    n = _ids(seq_ids, pos)
    _c_int("layer", layer)
    _c_int("n_select", n_select)
    _c_int("n_sink", n_sink)
    _c_int("n_recent", n_recent)
    ldq = _rows("q", q, n, _NH * _HD, (torch.bfloat16,))
    if out is None:
        out = torch.empty((n, _NKV, max(n_select, 0)), dtype=torch.int32, device=q.device)
    elif tuple(out.shape) != (n, _NKV, n_select) or out.dtype != torch.int32 or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous int32 tensor [{n}, 8, {n_select}]")
    st = _stream(cache, q, seq_ids, pos, out)
    check(lib().n550_kv8_select_blocks(st, q.data_ptr(), ldq, cache._ref, layer, seq_ids.data_ptr(),
                                       pos.data_ptr(), n, n_select, n_sink, n_recent, out.data_ptr()),
          "n550_kv8_select_blocks")
    return out
