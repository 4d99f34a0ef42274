"""The 8-bit KV cache without a GPU: argument checks of its entry points, which
run before any CUDA call, and the oracle's own e4m3 rounding."""
import ctypes as C

import pytest
import torch

import n550_qwen3_bringup_handover_b200 as n5
from kv8_oracle import POS, round_codes, scale_for, values


def struct(**kw):
    c = dict(k=4096, v=8192, k_scale=4096, v_scale=4096, k_bounds=4096, n_slots=2, n_layers=3, max_len=100)
    c.update(kw)
    return n5.KV8CacheStruct(*[c[f] for f, _ in n5.KV8CacheStruct._fields_])


P = 4096      # a well aligned address that is never read: every call below is refused first


def calls(L, cache, layer=0, ptr=P, ld=2048, n=1, rows=4):
    """Every entry point with otherwise good arguments."""
    r = C.byref(cache) if cache is not None else None
    return {
        "append": L.n550_kv8_append(None, r, layer, ptr, ptr, n5.BF16, ld, P, P, n, rows),
        "decode": L.n550_attention_decode_kv8(None, ptr, ld, r, layer, P, P, n, ptr, ld, None, 0),
        "sparse": L.n550_attention_sparse_kv8(None, ptr, ld, r, layer, P, P, P, 2, n, ptr, ld, None, 0),
        "prefill": L.n550_attention_prefill_kv8(None, ptr, ld, r, layer, P, n, rows, 0, ptr, ld, None, 0),
        "select": L.n550_kv8_select_blocks(None, ptr, ld, r, layer, P, P, n, 4, 1, 1, P),
    }


@pytest.mark.parametrize("bad", [
    dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=4104), dict(v=4097),
    dict(k_bounds=4100), dict(k_scale=4098), dict(n_slots=0), dict(n_layers=0), dict(max_len=0), dict(max_len=-5), dict(max_len=(1 << 30) + 1),
    dict(n_slots=1 << 20, n_layers=1 << 10),
])
def test_bad_caches_are_refused(bad):
    for name, rc in calls(n5.lib(), struct(**bad)).items():
        assert rc == n5.ERR_ARG, name


def test_bad_calls_are_refused():
    L = n5.lib()
    for kw in [dict(cache=None), dict(cache=struct(), layer=3), dict(cache=struct(), layer=-1),
               dict(cache=struct(), ptr=None), dict(cache=struct(), ptr=P + 8), dict(cache=struct(), ld=1000),
               dict(cache=struct(), ld=2052), dict(cache=struct(), n=-1), dict(cache=struct(), n=65536)]:
        for name, rc in calls(L, **kw).items():
            assert rc == n5.ERR_ARG, (name, kw)
    c = C.byref(struct())
    # append: element type, negative and too many rows
    assert L.n550_kv8_append(None, c, 0, P, P, 7, 1024, P, P, 1, 1) == n5.ERR_ARG
    assert L.n550_kv8_append(None, c, 0, P, P, n5.F32, 1024, P, P, 1, -1) == n5.ERR_ARG
    assert L.n550_kv8_append(None, c, 0, P, P, n5.F32, 1024, P, P, 1, 101) == n5.ERR_ARG
    # prefill: positions outside the cache
    assert L.n550_attention_prefill_kv8(None, P, 2048, c, 0, P, 1, 4, 97, P, 2048, None, 0) == n5.ERR_ARG
    assert L.n550_attention_prefill_kv8(None, P, 2048, c, 0, P, 1, 4, -1, P, 2048, None, 0) == n5.ERR_ARG
    assert L.n550_attention_prefill_kv8(None, P, 2048, c, 0, P, 1, 4, 2147483647, P, 2048, None, 0) == n5.ERR_ARG
    # sparse: a negative list length
    assert L.n550_attention_sparse_kv8(None, P, 2048, c, 0, P, P, P, -1, 1, P, 2048, None, 0) == n5.ERR_ARG
    assert L.n550_attention_sparse_kv8(None, P, 2048, c, 0, P, P, P, (1 << 24) + 1, 1, P, 2048, None, 0) == n5.ERR_ARG
    assert L.n550_attention_sparse_kv8(None, P, 2048, c, 0, P, P, None, 2, 1, P, 2048, None, 0) == n5.ERR_ARG
    # select: counts, a cache without bounds, too long a cache
    for n_select, sink, recent in [(0, 0, 0), (4, 3, 2), (4, -1, 2), (4, 1, -1), (4, 2147483647, 2147483647)]:
        assert L.n550_kv8_select_blocks(None, P, 2048, c, 0, P, P, 1, n_select, sink, recent, P) == n5.ERR_ARG
    nob = C.byref(struct(k_bounds=None))
    assert L.n550_kv8_select_blocks(None, P, 2048, nob, 0, P, P, 1, 4, 1, 1, P) == n5.ERR_ARG
    long = C.byref(struct(max_len=(n5.KV8_SELECT_MAX_BLOCKS + 1) * 64))
    assert L.n550_kv8_select_blocks(None, P, 2048, long, 0, P, P, 1, 4, 1, 1, P) == n5.ERR_UNSUPPORTED


def test_empty_calls_do_nothing():
    L, c = n5.lib(), struct()
    for name, rc in calls(L, c, n=0).items():
        assert rc == n5.OK, name
    r = C.byref(c)
    assert L.n550_kv8_append(None, r, 0, None, None, n5.F32, 1024, None, None, 5, 0) == n5.OK
    assert L.n550_attention_prefill_kv8(None, None, 2048, r, 0, None, 5, 0, 0, None, 2048, None, 0) == n5.OK
    assert L.n550_attention_kv8_workspace(0) == 0
    assert L.n550_attention_prefill_kv8_workspace(0, 4, 0) == 0


def test_workspace_covers_every_pass():
    """A call of L queries may end with a pass of any smaller number, whose instance
    has more runs: the workspace never shrinks with L."""
    L = n5.lib()
    sizes = [L.n550_attention_prefill_kv8_workspace(1, q, 100000) for q in range(1, 9)]
    assert sizes == sorted(sizes) and sizes[0] == L.n550_attention_kv8_workspace(1)
    # 296 runs of 4 queries: two partials of 8 columns x (128 + max + sum) and a record each
    assert sizes[7] >= 296 * (2 * 8 * 130 * 4 + 16)
    # many queries over a context that the passes would read too often: the context as BF16
    assert L.n550_attention_prefill_kv8_workspace(3, 512, 88) == 3 * 600 * 4096


def test_cache_class_refuses_tensors():
    with pytest.raises(ValueError):
        n5.KV8Cache(0, 64)
    with pytest.raises(ValueError):
        n5.KV8Cache()
    z = torch.zeros((1, 1, 8, 64, 128)).to(torch.float8_e4m3fn)
    s = torch.zeros((1, 1, 8, 1))
    with pytest.raises(ValueError):                       # not on a GPU
        n5.KV8Cache(k=z, v=z, k_scale=s, v_scale=s)
    with pytest.raises(ValueError):                       # a part is missing
        n5.KV8Cache(k=z, v=z, k_scale=s)
    with pytest.raises(ValueError):                       # scales of another shape
        n5.KV8Cache(k=z, v=z, k_scale=s, v_scale=torch.zeros((1, 1, 8, 2)))


def test_oracle_rounding_is_e4m3():
    """Every code's value, and rounding against torch's own conversion where that
    is defined (finite values up to 448)."""
    codes = torch.arange(256, dtype=torch.int64).to(torch.uint8)
    v = codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(values(codes).nan_to_num(nan=999.0), v.nan_to_num(nan=999.0))
    g = torch.Generator().manual_seed(3)
    x = torch.cat([torch.randn(4000, generator=g) * 2.0 ** e for e in range(-12, 7)]).clamp(-448, 448)
    mid = ((POS[1:] + POS[:-1]) / 2).float()              # ties
    x = torch.cat([x, mid, -mid, POS.float()])
    assert torch.equal(round_codes(x.double()), x.to(torch.float8_e4m3fn).view(torch.uint8))
    assert scale_for(torch.tensor([448.0])) == 1.0 and scale_for(torch.tensor([448.5])) == 2.0
    assert scale_for(torch.tensor([0.0])) == 2.0 ** -126


def test_merge_check_refuses():
    """No workspace, too small or unaligned a one, no sequences, no rows to write to."""
    L = n5.lib()
    need = L.n550_attention_kv8_workspace(1)
    for n, ws, size, out, ld in [(1, None, need, P, 2048), (1, P, need - 1, P, 2048), (1, P + 8, need, P, 2048), (0, P, need, P, 2048),
                                 (65536, P, need, P, 2048), (1, P, need, None, 2048), (1, P, need, P, 2040)]:
        assert L.n550_check_kv8_merge(None, n, ws, size, out, ld) == n5.ERR_ARG


def test_wrappers_refuse_numbers_beyond_a_c_int():
    """ctypes passes the lower 32 bits of an int: layer 2^32 would be layer 0, and rows
    2^32 + 2048 elements apart would be read 2048 apart."""
    ids, q = torch.zeros(2, dtype=torch.int32), torch.zeros((2, 2048), dtype=torch.bfloat16)
    kv, blocks = torch.zeros((2, 1024)), torch.zeros((2, 8, 1), dtype=torch.int32)
    for big in (2 ** 31, 2 ** 32, 2 ** 32 + 1, -2 ** 32, 2 ** 64):
        calls = [lambda: n5.kv8_append(None, kv, kv, ids, ids, 1, big),
                 lambda: n5.attention_decode_kv8(q, None, ids, ids, big),
                 lambda: n5.attention_sparse_kv8(q, None, ids, ids, blocks, big),
                 lambda: n5.attention_prefill_kv8(q, None, ids, 1, 0, big),
                 lambda: n5.attention_prefill_kv8(q, None, ids, 1, big, 0),
                 lambda: n5.kv8_select_blocks(q, None, ids, ids, big, 4),
                 lambda: n5.kv8_select_blocks(q, None, ids, ids, 0, 4, big, 0),
                 lambda: n5.kv8_select_blocks(q, None, ids, ids, 0, 4, 0, big)]
        for call in calls:
            with pytest.raises(ValueError, match="32 bits"):
                call()
    far = torch.empty_strided((2, 2048), (2 ** 32 + 2048, 1), dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="row stride"):
        n5.attention_decode_kv8(far, None, ids, ids, 0)
    with pytest.raises(ValueError, match="row stride"):
        n5.attention_decode_kv8(q, None, ids, ids, 0, out=far)


def test_exact_mode_with_the_8_bit_cache_is_refused():
    h = C.c_void_p()
    for mode, want in [(n5.MODE_EXACT | n5.MODEL_KV8, n5.ERR_UNSUPPORTED), (7, n5.ERR_ARG), (7 | n5.MODEL_KV8, n5.ERR_ARG),
                       (n5.MODE_FAST | 2 * n5.MODEL_KV8, n5.ERR_ARG), (-1, n5.ERR_ARG)]:
        cfg = n5.ModelConfig(1, 64, 16, mode, 16)
        assert n5.lib().n550_qwen3_init_random(C.byref(h), 0, 0.02, C.byref(cfg)) == want
        assert not h


def test_values_are_bf16_numbers_for_scales_in_range():
    """Every code times 2^-124 .. 2^119 (and neither 2^-125 nor 2^120) is a finite BF16 number."""
    v = values(torch.arange(256).to(torch.uint8))
    v = v[~v.isnan()]

    def whole(e):
        x = v * 2.0 ** e
        return torch.equal(x.to(torch.float32).to(torch.bfloat16).double(), x)

    assert all(whole(e) for e in range(-124, 120))
    assert not whole(-125) and not whole(120)
    # the smallest scale that append gives blocks at the statement's borders
    assert scale_for(torch.tensor([448.0 * 2.0 ** -125], dtype=torch.float64)) == 2.0 ** -125
    assert scale_for(torch.tensor([448.0 * 2.0 ** 119], dtype=torch.float64)) == 2.0 ** 119
    assert scale_for(torch.tensor([448.5 * 2.0 ** 119], dtype=torch.float64)) == 2.0 ** 120
