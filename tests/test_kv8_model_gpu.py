"""The model runtime over the 8-bit KV cache (n550_qwen3_use_kv8): its cache holds
what the definitions give for the model's own K and V, and its decode, prefill
and graph routes agree with one another.

Logits of two routes (GEMMs that sum in another order) differ by more than with the
BF16 cache: a K or V row that differs in the last bit of its BF16 form (2^-8 of the
value) falls on the other side of an e4m3 rounding border (2^-3 of the value apart)
in up to 2^-5 of its elements, and those move by one step, up to 2^-3 of the value:
sqrt(2^-5) * 2^-3 = 2.2 % in the mean square of every layer's attention, so at most
that of the residual stream it is a part of, and of the logits, whose largest error
is to their largest value as their mean squares are (both are the extremes of 151936
nearly normal values). TOL is that with room for the 3e-3 of the BF16 roundings."""
import numpy as np
import pytest
import torch

import n550_qwen3_bringup_handover_b200 as n5
import oracle
from kv8_oracle import BLOCK

pytestmark = pytest.mark.gpu
TOL = 2.5e-2


def toks(n, seed):
    return torch.from_numpy(oracle.synth_tokens(n, seed, 0x544F4B)).cuda()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def model(cuda):
    m = n5.Model(seed=0, max_seqs=40, max_len=300, max_tokens=1300, kv8=True)
    yield m
    m.close()


def rel(a, b):
    return float((a - b).abs().max() / b.abs().max())


def logits(n):
    return torch.empty((n, 151936), dtype=torch.float32, device="cuda")


def layer0_kv(m, tokens):
    """K and V rows of layer 0 (FP32, [n, 8, 128]) from the library's own ops."""
    bits = lambda i, *s: torch.from_numpy(m.weight_bits(i).view(np.int16)).view(torch.bfloat16).cuda().view(*s)  # noqa: E731
    x = bits(0, 151936, 1024)[tokens.long()].float()
    xb = n5.rmsnorm(x, bits(1, 1024), out_dtype=torch.bfloat16)
    k = n5.gemm(xb, bits(3, 1024, 1024)).view(-1, 128)
    v = n5.gemm(xb, bits(4, 1024, 1024))
    k = n5.rmsnorm(k, bits(6, 128)).view(-1, 1024)
    return n5.rope(k.contiguous(), 8, 0).view(-1, 8, 128), v.view(-1, 8, 128)


def check_layer0(m, tokens, slot):
    """Codes times scales of layer 0 against the rows: half an e4m3 step (2^-4 of the
    value, 2^-10 of the scale below 2^-6) and the BF16 rounding before it (2^-8),
    with 2^-12 of slack for sums in another order."""
    c = m.kv8_cache()
    n = len(tokens)
    b = torch.arange(n, device="cuda") // BLOCK
    for rows, codes, scale in zip(layer0_kv(m, tokens), (c.k, c.v), (c.k_scale, c.v_scale)):
        s = scale[slot, 0][:, b, None]
        got = (codes[slot, 0, :, :n].float() * s).transpose(0, 1)
        tol = rows.abs() * (2.0 ** -4 + 2.0 ** -8 + 2.0 ** -12) + s.transpose(0, 1) * 2.0 ** -10 + 1e-6
        assert ((got - rows).abs() <= tol).all()


@pytest.mark.parametrize("n", [1, 3, 40, 290])
def test_cache_holds_the_layers_rows(model, n):
    t = toks(n, 5)
    model.prefill(t.view(1, n), i32([7]), 0, next_token=i32([0]))
    check_layer0(model, t, 7)


@pytest.mark.parametrize("n_seqs,L", [(4, 260), (5, 259), (9, 3), (64, 1)])
def test_cache_of_a_batch(cuda, n_seqs, L):
    """Rows written by the epilogues of the tile GEMM (from 1024 rows) and of the
    weight-streaming one, in slots out of order; the other slots stay empty."""
    m = n5.Model(seed=0, max_seqs=66, max_len=270, max_tokens=1300, kv8=True)
    try:
        t = toks(n_seqs * L, 7).view(n_seqs, L)
        ids = torch.randperm(66, generator=torch.Generator().manual_seed(L))[:n_seqs].to(torch.int32)
        m.prefill(t, ids.cuda(), 0, next_token=torch.empty(n_seqs, dtype=torch.int32, device="cuda"))
        for s in range(n_seqs):
            check_layer0(m, t[s], int(ids[s]))
        rest = torch.ones(66, dtype=torch.bool)
        rest[ids.long()] = False
        c = m.kv8_cache()
        assert not c.k.view(torch.uint8)[rest.cuda()].any() and not c.v.view(torch.uint8)[rest.cuda()].any()
        assert n5.device_status() == n5.OK
    finally:
        m.close()


@pytest.mark.parametrize("n_seqs", [1, 4, 6, 20, 36])
def test_decode_agrees_with_prefill(model, n_seqs):
    """Token n decoded after a prefill of n, and n + 1 tokens prefilled: every
    decode route (GEMV, weight-streaming, split) against the prefill's."""
    n = 70
    t = toks(n_seqs * (n + 1), 11).view(n_seqs, n + 1)
    ids = torch.randperm(40, generator=torch.Generator().manual_seed(n_seqs))[:n_seqs].to(torch.int32).cuda()
    want, got = logits(n_seqs), logits(n_seqs)
    model.prefill(t.contiguous(), ids, 0, want)
    model.prefill(t[:, :n].contiguous(), ids, 0, next_token=torch.empty(n_seqs, dtype=torch.int32, device="cuda"))
    model.decode(t[:, n].contiguous(), ids, i32([n] * n_seqs), got)
    torch.cuda.synchronize()
    assert n5.device_status() == n5.OK
    assert rel(got, want) <= TOL


@pytest.mark.parametrize("n_seqs", [1, 8, 20, 70])
def test_appending_in_the_kernel_before_is_bit_identical(cuda, n_seqs):
    """Decode steps over several blocks from ragged positions (one of them 0, one the
    cache's last): ids, codes, scales and bounds of both ways of appending."""
    steps, max_len = 70, 260
    start = [(s * 37) % 150 for s in range(n_seqs)]
    t = toks(n_seqs * 150, 61).view(n_seqs, 150)
    got = []
    m = n5.Model(seed=0, max_seqs=n_seqs, max_len=max_len, max_tokens=256, kv8=True)
    try:
        for fused in (1, 0):
            n5.check(n5.lib().n550_qwen3_fused_attention_prep(fused))
            c = m.kv8_cache()
            for x in (c.k, c.v, c.k_bounds):
                x.view(torch.uint8).zero_()
            for s in range(n_seqs):
                if start[s]:
                    m.prefill(t[s:s + 1, :start[s]].contiguous(), i32([s]), 0, next_token=i32([0]))
            tok, out = t[:, 149].clone(), torch.empty((steps, n_seqs), dtype=torch.int32, device="cuda")
            m.decode_steps(tok, torch.arange(n_seqs, dtype=torch.int32, device="cuda"), i32(start), steps, out, use_graph=False)
            last = i32([max_len - 1])                           # (a context with holes: only its row matters)
            m.decode(t[0, :1].contiguous(), i32([n_seqs - 1]), last, next_token=i32([0]))
            torch.cuda.synchronize()
            end = [p + steps for p in start]
            nb = [-(-e // BLOCK) for e in end]
            got.append([out.clone()] + [x[s, :, :, :end[s]].view(torch.uint8).clone() for x in (c.k, c.v) for s in range(n_seqs)] +
                       [x[s, :, :, :nb[s]].clone() for x in (c.k_scale, c.v_scale, c.k_bounds.view(torch.uint8))
                        for s in range(n_seqs)] +
                       [x[n_seqs - 1, 0, :, max_len - 1].view(torch.uint8).clone() for x in (c.k, c.v)])
    finally:
        n5.lib().n550_qwen3_fused_attention_prep(1)
        m.close()
    assert n5.device_status() == n5.OK
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_chunked_prefill_and_rows(model):
    """A prompt in chunks (whole-tile and few-query attention) against the whole, and
    all-row logits of drafted tokens against single decodes."""
    t = toks(200, 21)
    nx = i32([0])
    want, got = logits(1), logits(1)
    model.prefill(t.view(1, 200), i32([3]), 0, want, nx)
    for at, L in ((0, 150), (150, 43), (193, 7)):
        model.prefill(t[at:at + L].view(1, L).contiguous(), i32([9]), at, got, nx)
    assert rel(got, want) <= TOL
    _, rows = model.forward_rows(t[:100].cpu().numpy(), 0, want_logits=True)
    for L in (5, 12):
        _, rows = model.forward_rows(t[100:100 + L].cpu().numpy(), 100, want_logits=True)
        one = logits(1)
        for j in range(L):
            model.decode(t[100 + j:101 + j].contiguous(), i32([0]), i32([100 + j]), one)
            assert rel(torch.from_numpy(rows[j]).cuda(), one[0]) <= TOL


def test_grouped_prefill(cuda):
    """More contexts than the BF16 copy holds at once: same logits as one at a time."""
    m = n5.Model(seed=0, max_seqs=9, max_len=16384, max_tokens=9 * 20, kv8=True)   # 4 contexts of 16384 positions
    try:
        n, p0 = 9, 16000
        t = toks(n * 20, 31).view(n, 20)
        ids = i32(list(range(n)))
        all_, one = logits(n), logits(1)
        m.prefill(t.contiguous(), ids, p0, all_)
        for s in (0, 4, 8):
            m.prefill(t[s:s + 1].contiguous(), ids[s:s + 1].contiguous(), p0, one)
            assert rel(all_[s], one[0]) <= TOL
        # two prompts in an order that differs from group to group: equal rows, bit for bit
        kind = torch.tensor([0, 1, 1, 0, 1, 0, 0, 1, 0], device="cuda")
        m.prefill(t[:2][kind].contiguous(), ids, p0, all_)
        assert torch.equal(all_, all_[:2][kind]) and not torch.equal(all_[0], all_[1])
    finally:
        m.close()


def test_graph_replay_switching_back_and_refusals(cuda):
    m = n5.Model(seed=0, max_seqs=6, max_len=128, max_tokens=256)
    try:
        with pytest.raises(n5.N550Error):
            m.kv8_cache()
        t = toks(5 * 30, 41).view(5, 30)
        ids = i32([4, 0, 3, 1, 2])

        def generate(graph):
            nx, out = torch.empty(5, dtype=torch.int32, device="cuda"), torch.empty((20, 5), dtype=torch.int32, device="cuda")
            m.prefill(t, ids, 0, next_token=nx)
            m.decode_steps(nx, ids, i32([30] * 5), 20, out, use_graph=graph)
            torch.cuda.synchronize()
            return out

        plain = generate(True)
        m.use_kv8()
        a, b, c = generate(False), generate(True), generate(True)
        assert torch.equal(a, b) and torch.equal(a, c)
        with pytest.raises(n5.N550Error):
            m.forward_dump(np.arange(4, dtype=np.int32), 0)
        m.use_kv8(False)
        assert torch.equal(generate(True), plain)
    finally:
        m.close()
    e = n5.Model(seed=0, max_seqs=1, max_len=64, max_tokens=16, gemm_mode=n5.MODE_EXACT)
    try:
        with pytest.raises(n5.N550Error):
            e.use_kv8()
    finally:
        e.close()


def test_no_room_for_the_cache_to_go_back_to(cuda):
    """The BF16 cache (twice the 8-bit one) does not fit any more: N550_ERR_OOM from there
    on, not a launch over memory that is gone, and a second try that has room works."""
    m = n5.Model(seed=0, max_seqs=1, max_len=32768, max_tokens=64, kv8=True)       # BF16 3.8 GB, 8-bit 1.9 GB
    hold = None
    try:
        t, ids, nx = toks(20, 71), i32([0]), i32([0])
        want, got = logits(1), logits(1)
        m.use_kv8(False)
        m.prefill(t.view(1, 20), ids, 0, want, nx)
        m.use_kv8()
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        free = torch.cuda.mem_get_info()[0]
        hold = torch.empty(free - (512 << 20), dtype=torch.uint8, device="cuda")
        calls = [lambda: m.use_kv8(False), lambda: m.prefill(t.view(1, 20), ids, 0, got, nx),
                 lambda: m.decode(nx, ids, i32([20]), got), lambda: m.forward_batch(np.arange(4, dtype=np.int32), 0),
                 lambda: m.forward_rows(np.arange(4, dtype=np.int32), 0),
                 lambda: m.decode_steps(nx, ids, i32([20]), 2, torch.empty((2, 1), dtype=torch.int32, device="cuda"))]
        for call in calls:
            with pytest.raises(n5.N550Error) as e:
                call()
            assert e.value.status == n5.ERR_OOM
        with pytest.raises(n5.N550Error):
            m.kv8_cache()
        hold = None
        torch.cuda.empty_cache()
        m.use_kv8(False)
        m.prefill(t.view(1, 20), ids, 0, got, nx)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    finally:
        hold = None
        m.close()
        torch.cuda.empty_cache()


def test_a_model_that_does_not_fit_leaves_no_error_behind(cuda):
    """229 GB of BF16 cache: N550_ERR_OOM, and the next model is built and runs."""
    torch.cuda.empty_cache()
    for _ in range(2):
        with pytest.raises(n5.N550Error) as e:
            n5.Model(seed=0, max_seqs=1, max_len=2_000_000, max_tokens=16)
        assert e.value.status == n5.ERR_OOM
        m = n5.Model(seed=0, max_seqs=1, max_len=64, max_tokens=16)
        try:
            assert m.forward_batch(np.arange(4, dtype=np.int32), 0)[0] >= 0
        finally:
            m.close()


def test_a_cache_that_fits_in_8_bits_alone(cuda):
    """115 GB of codes where the BF16 cache would be 229 GB: the model is created with it, its
    steps are those of a small model, and there is no way to BF16 from it."""
    import ctypes as C
    torch.cuda.empty_cache()
    t, ids = toks(21, 81), i32([0])
    got = []
    for max_len in (64, 2_000_000):
        m = n5.Model(seed=0, max_seqs=1, max_len=max_len, max_tokens=64, kv8=True)
        try:
            cfg = n5.ModelConfig()
            n5.check(n5.lib().n550_qwen3_get_config(m.handle, C.byref(cfg)))
            assert cfg.gemm_mode == n5.MODE_FAST | n5.MODEL_KV8 and cfg.max_len == max_len

            def step():
                a, b = logits(1), logits(1)
                m.prefill(t[:20].view(1, 20), ids, 0, a)
                m.decode(t[20:], ids, i32([20]), b)
                torch.cuda.synchronize()
                return [a, b]

            got.append(step())
            if max_len > 64:
                with pytest.raises(n5.N550Error) as e:
                    m.use_kv8(False)
                assert e.value.status == n5.ERR_OOM
                m.use_kv8()
                got.append(step())
        finally:
            m.close()
    assert n5.device_status() == n5.OK
    for x in got[1:]:
        assert torch.equal(x[0], got[0][0]) and torch.equal(x[1], got[0][1])


def test_the_cache_of_a_model_on_another_device_is_refused(model, monkeypatch):
    """torch copies memory of another device to the current one: appends to such a
    copy would be lost. (Here a copy on the same device stands in for it.)"""
    assert model.kv8_cache().k.data_ptr() == model.kv8_cache()._c.k
    was = torch.as_tensor
    monkeypatch.setattr(torch, "as_tensor", lambda *a, **kw: was(*a, **kw).clone())
    with pytest.raises(ValueError, match="another device"):
        model.kv8_cache()
