"""The 8-bit KV cache on the GPU against the binary64 definitions of
kv8_oracle.py: append bit for bit, selections index for index, attention within
the roundings it makes.

Attention tolerance, per element: the output is rounded to BF16 (2^-8 |out|);
the softmax weights enter the tensor cores in FP16's 11 bits (2^-12 each; the
allowance is 2^-11) or, on the whole-tile prefill route, in BF16 (2^-8 each), and small ones as
multiples of 2^-25 of the largest, which moves the result by at most that part of
mass (Cache.attend); sums and scores in FP32 and the hardware exponential add less
than 2^-13 of mass at these sizes (score errors below 2^-15: 128 products of
magnitude <= 2^5 summed with 2^-24 each)."""
import pytest
import torch

import n550_qwen3_bringup_handover_b200 as n5
from kv8_oracle import BLOCK, Cache

pytestmark = pytest.mark.gpu

HALF, BF = 2.0 ** -11 + 2.0 ** -13, 2.0 ** -8 + 2.0 ** -13


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rows(n, cols, dtype, seed, scale=1.0):
    return (torch.randn((n, cols), generator=gen(seed)) * scale).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def fresh(n_slots, max_len, n_layers=2, fill=0x7F, bounds=True):
    """A cache whose memory holds NaN codes and NaN scales everywhere."""
    c = n5.KV8Cache(n_slots, max_len, n_layers=n_layers, bounds=bounds)
    for t in (c.k, c.v, c.k_bounds):
        if t is not None:
            t.view(torch.uint8).fill_(fill)
    c.k_scale.fill_(float("nan"))
    c.v_scale.fill_(float("nan"))
    return c


def filled(n_slots, max_len, seed, layer=1, lengths=None, kscale=1.0):
    """A cache with lengths[slot] appended positions (all: max_len) per slot and its oracle copy."""
    c = fresh(n_slots, max_len)
    for s in range(n_slots):
        L = max_len if lengths is None else lengths[s]
        if L:
            k = rows(L, 1024, torch.float32, seed + 2 * s, kscale).cuda()
            v = rows(L, 1024, torch.float32, seed + 2 * s + 1).cuda()
            n5.kv8_append(c, k, v, i32([s]), i32([0]), L, layer)
    return c, Cache.of(c, layer)


def assert_state(c, ref, layer):
    got = Cache.of(c, layer)
    for w in "kv":
        assert torch.equal(got.code[w], ref.code[w]), w
        assert torch.equal(got.scale[w].nan_to_num(nan=-1), ref.scale[w].nan_to_num(nan=-1)), w
    # as values: min and max of a channel with both zeros may have either's sign
    assert torch.equal(torch.where(got.bounds == 128, 0, got.bounds), torch.where(ref.bounds == 128, 0, ref.bounds))


def assert_near(out, ref, mass, weight=HALF):
    o = out.double().cpu()
    assert torch.isfinite(o).all()
    err, tol = (o - ref).abs(), 2.0 ** -8 * ref.abs() + weight * mass
    assert (err <= tol).all(), f"{int((err > tol).sum())} of {err.numel()} off, worst {(err - tol).max():.3g} over"


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L,pos,max_len", [
    (1, [0, 63, 64, 130, 5], 200),        # single tokens: a block's first, last, another's
    (7, [0, 60, 120, 193, 1], 200),       # across a border, to the very end
    (64, [0, 64, 1, 136, 63], 200),       # whole and shifted blocks
    (150, [0, 50, 13, 49, 37], 200),      # several blocks
    (200, [0, 0, 0, 0, 0], 200),          # the whole slot, whose last block is short
])
def test_append_matches_definition(dtype, L, pos, max_len):
    c = fresh(6, max_len)
    base_k, base_v = rows(6 * max_len, 1024, dtype, 1, 0.7), rows(6 * max_len, 1024, dtype, 2)
    n5.kv8_append(c, base_k.cuda(), base_v.cuda(), i32(range(6)), i32([0] * 6), max_len, 1)
    ref = fresh_ref = Cache.of(fresh(6, max_len), 1)
    ref.append(base_k, base_v, list(range(6)), [0] * 6, max_len)
    assert_state(c, fresh_ref, 1)
    ids = [4, 0, 5, 2, 1]                                   # slot 3 is left alone
    k, v = rows(5 * L, 1024, dtype, 3, 2.0), rows(5 * L, 1024, dtype, 4, 0.01)
    n5.kv8_append(c, k.cuda(), v.cuda(), i32(ids), i32(pos), L, 1)
    ref.append(k, v, ids, pos, L)
    assert_state(c, ref, 1)
    assert (c.k[:, 0].view(torch.uint8) == 0x7F).all()      # the other layer


def test_append_token_by_token_with_growing_and_shrinking_values():
    """130 single tokens whose size jumps by powers of two: scales grow inside a
    block and never shrink, held codes are rounded anew, down to zero."""
    c, ref = fresh(2, 140), Cache.of(fresh(2, 140), 0)
    for t in range(130):
        size = 2.0 ** ((t * 7) % 23 - 11)
        k, v = rows(2, 1024, torch.float32, 100 + t, size), rows(2, 1024, torch.float32, 300 + t, 1 / size)
        n5.kv8_append(c, k.cuda(), v.cuda(), i32([1, 0]), i32([t, t]), 1, 0)
        ref.append(k, v, [1, 0], [t, t], 1)
    assert_state(c, ref, 0)


def test_append_rewound_and_reused_slots():
    c, ref = fresh(1, 300), Cache.of(fresh(1, 300), 1)
    for i, (p, L, size) in enumerate([(0, 200, 5.0), (130, 3, 0.1), (133, 60, 1.0), (0, 10, 0.5), (10, 1, 90.0)]):
        k, v = rows(L, 1024, torch.bfloat16, 10 + i, size), rows(L, 1024, torch.bfloat16, 50 + i, size)
        n5.kv8_append(c, k.cuda(), v.cuda(), i32([0]), i32([p]), L, 1)
        ref.append(k, v, [0], [p], L)
        assert_state(c, ref, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [20, 6])
def test_append_special_values(L, dtype):
    inf, nan = float("inf"), float("nan")
    k = rows(20, 1024, torch.float32, 8)
    k[0, 0], k[1, 1], k[2, 2], k[3, 3] = inf, -inf, nan, 3.3e38
    k[:, 128:256] = 0.0                                     # a head of zeros
    k[:, 256:384] *= 1e-41                                  # subnormal numbers
    k[:, 384:512] = nan                                     # nothing but NaN
    k[:, 512:640] = inf                                     # nothing but infinities
    k[5, 640:768] = 448.0 * 2 ** 9                          # the border of a scale, and just over it
    k[5, 768:896] = torch.nextafter(torch.tensor(448.0 * 2 ** 9), torch.tensor(inf))
    k = k[:L].to(dtype)
    v = -k.flip(1)
    for p in (0, 30):
        c, ref = fresh(1, 64), Cache.of(fresh(1, 64), 0)
        if p:
            z = rows(30, 1024, torch.float32, 9)
            n5.kv8_append(c, z.cuda(), z.cuda(), i32([0]), i32([0]), 30, 0)
            ref.append(z, z, [0], [0], 30)
        n5.kv8_append(c, k.cuda(), v.cuda(), i32([0]), i32([p]), L, 0)
        ref.append(k, v, [0], [p], L)
        assert_state(c, ref, 0)


def test_append_skips_what_does_not_fit_and_takes_strided_rows():
    c, ref = filled(3, 100, 11)                             # (a block's held positions must have been appended)
    was = Cache.of(c, 1).code["k"]
    ids, pos = [0, 3, -1, 1, 2, 2147483647], [95, 0, 0, -1, 94, 2]
    wide = rows(6 * 6, 3 * 1024, torch.bfloat16, 12)
    dev = wide.cuda()
    n5.kv8_append(c, dev[:, 1024:2048], dev[:, 2048:], i32(ids), i32(pos), 6, 1)
    ref.append(wide[:, 1024:2048], wide[:, 2048:], ids, pos, 6)   # only slot 2 fits
    assert_state(c, ref, 1)
    assert torch.equal(ref.code["k"][:2], was[:2]) and not torch.equal(ref.code["k"][2], was[2])
    a, b = fresh(3, 100), fresh(3, 100, bounds=False)       # a cache without bounds
    for x in (a, b):
        n5.kv8_append(x, dev[:18, 1024:2048], dev[:18, 2048:], i32([1, 0, 2]), i32([0, 64, 0]), 6, 1)
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8))
    assert torch.equal(a.k_scale.nan_to_num(nan=-1), b.k_scale.nan_to_num(nan=-1))


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("pos", [
    [0], [63], [64], [299], [-1],
    [299, 0, 1, 62, 63, 64, 65, 127, 128, -1, 200],
    [5] * 40,
])
def test_decode_matches_definition(pos, split):
    n = len(pos)
    c, ref = filled(3, 300, 20)
    ids = [(2 * i + 1) % 3 for i in range(n)]               # slots shared by sequences
    q = rows(n, 2048, torch.bfloat16, 21)
    out = n5.attention_decode_kv8(q.cuda(), c, i32(ids), i32(pos), 1, split=split)
    assert_near(out, *ref.attend(q, ids, pos))
    assert n5.device_status() == n5.OK


def test_decode_ignores_what_lies_behind_the_context():
    """NaN codes and NaN scales behind every context, in its last block too."""
    lengths = [0, 1, 64, 70, 129]
    c, ref = filled(5, 200, 40, lengths=lengths)
    q = rows(5, 2048, torch.bfloat16, 41)
    pos = [n - 1 for n in lengths]
    for split in (True, False):
        out = n5.attention_decode_kv8(q.cuda(), c, i32(range(5)), i32(pos), 1, split=split)
        assert_near(out, *ref.attend(q, list(range(5)), pos))
        assert (out[0] == 0).all()


@pytest.mark.parametrize("qscale,kscale", [(30.0, 1.0), (1e30, 1e-30), (1e-30, 1e30), (0.0, 1.0)])
def test_decode_ranges(qscale, kscale):
    """Peaked scores, and queries and keys at the far ends of the exponent range."""
    c, ref = filled(2, 190, 60, kscale=kscale)
    q = rows(2, 2048, torch.bfloat16, 61, qscale)
    out = n5.attention_decode_kv8(q.cuda(), c, i32([1, 0]), i32([189, 100]), 1)
    want, mass = ref.attend(q, [1, 0], [189, 100])
    # scores up to ~30 * 30: FP32 sums of 128 products err by up to 2^-24 * 128 * 2^10 = 2^-7
    assert_near(out, want, mass, HALF + (2.0 ** -7 if qscale == 30.0 else 0.0))


def test_decode_bad_slots_positions_and_strides():
    c, ref = filled(2, 150, 70)
    ids, pos = [-1, 2, 0, 1, 2147483647], [10, 10, 149, 2147483647, 3]
    wide = rows(5, 3000 * 8 // 8, torch.bfloat16, 71).cuda()
    buf = torch.full((7, 2560), 7.0, dtype=torch.bfloat16, device="cuda")
    n5.attention_decode_kv8(wide, c, i32(ids), i32(pos), 1, out=buf[:5])
    want, mass = ref.attend(wide[:, :2048].cpu(), ids, pos)
    assert_near(buf[:5, :2048], want, mass)
    assert (buf[:2, :2048] == 0).all() and (buf[4, :2048] == 0).all()
    assert (buf[:, 2048:] == 7).all() and (buf[5:] == 7).all()


def test_decode_ragged_long_contexts():
    """Contexts from one block to hundreds in one call, checked against a plain binary64 product on the GPU."""
    lens = [20000, 1, 700, 8191, 64]
    c = fresh(5, 20000, n_layers=1)
    for s, L in enumerate(lens):
        k, v = rows(L, 1024, torch.float32, 80 + s).cuda(), rows(L, 1024, torch.float32, 90 + s).cuda()
        n5.kv8_append(c, k, v, i32([s]), i32([0]), L, 0)
    q = rows(5, 2048, torch.bfloat16, 85).cuda()
    out = n5.attention_decode_kv8(q, c, i32(range(5)), i32([L - 1 for L in lens]), 0)
    for s, L in enumerate(lens):
        t = torch.arange(L, device="cuda") // BLOCK
        k = c.k[s, 0, :, :L].double() * c.k_scale[s, 0][:, t, None].double()
        v = c.v[s, 0, :, :L].double() * c.v_scale[s, 0][:, t, None].double()
        w = torch.softmax(q[s].double().view(8, 2, 128) @ k.transpose(1, 2) * 0.08838834764831845, -1)
        assert_near(out[s], (w @ v).view(-1).cpu(), (w @ v.abs()).view(-1).cpu())


@pytest.mark.parametrize("n", [33, 300, 700])
def test_decode_many_sequences(n):
    """More sequences than a warp, than one round of the run search, and than two;
    empty ones among them, also in rows and at both ends."""
    c, ref = filled(4, 210, 75)
    g = gen(n)
    pos = torch.randint(-1, 210, (n,), generator=g).tolist()
    pos[:9] = [-1] * 9
    pos[-4:] = [-1] * 4
    pos[20:31] = [-1] * 11
    ids = torch.randint(0, 4, (n,), generator=g).tolist()
    q = rows(n, 2048, torch.bfloat16, 76).cuda()
    a = n5.attention_decode_kv8(q, c, i32(ids), i32(pos), 1)
    b = n5.attention_decode_kv8(q, c, i32(ids), i32(pos), 1, split=False)
    some = sorted(set(torch.randint(0, n, (25,), generator=g).tolist()) | {0, 9, 25, n - 1, n - 5})
    for out in (a, b):
        assert_near(out[some], *ref.attend(q[some].cpu(), [ids[i] for i in some], [pos[i] for i in some]))
        assert (out[[i for i in range(n) if pos[i] < 0]] == 0).all()
    # split or not, a row differs by the order of its sums alone (two roundings to BF16)
    assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -9).all()


def test_decode_with_block_scales_far_apart():
    """V (and K) of each block in a magnitude of its own: tiles of one block, and an
    accumulator that changes its scale up and down."""
    max_len = 64 * 14 + 9
    g = gen(77)
    size = torch.exp2(torch.randint(-20, 21, (15,), generator=g).float()).repeat_interleave(64)[:max_len, None]
    c = fresh(1, max_len)
    k, v = rows(max_len, 1024, torch.float32, 78), rows(max_len, 1024, torch.float32, 79) * size
    n5.kv8_append(c, k.cuda(), v.cuda(), i32([0]), i32([0]), max_len, 1)
    ref = Cache.of(c, 1)
    q = rows(3, 2048, torch.bfloat16, 80, 2.0)
    pos = [max_len - 1, 500, 320]
    for split in (True, False):
        out = n5.attention_decode_kv8(q.cuda(), c, i32([0] * 3), i32(pos), 1, split=split)
        assert_near(out, *ref.attend(q, [0] * 3, pos, floor=2.0 ** -12))
    out = n5.attention_prefill_kv8(q[:3].cuda(), c, i32([0]), 3, 700, 1)
    assert_near(out, *ref.attend(q, [0], [700], 3, floor=2.0 ** -12))


def test_decode_nan_stays_in_its_place():
    c, ref = filled(1, 200, 82)
    v = c.v.view(torch.uint8)
    v[0, 1, 3, 77, 5] = 0x7F                                # V, KV head 3, position 77, dimension 5
    c.k.view(torch.uint8)[0, 1, 6, 150, 9] = 0xFF           # K, KV head 6, position 150
    q = rows(4, 2048, torch.bfloat16, 83)
    q[3, 128] = float("nan")                                # head 1 of the last query
    q[2, 0] = float("inf")                                  # head 0 of the third
    pos = [199, 76, 149, 199]
    out = n5.attention_decode_kv8(q.cuda(), c, i32([0] * 4), i32(pos), 1)
    bad = torch.zeros((4, 16, 128), dtype=torch.bool)
    bad[0, 6:8, 5] = bad[2, 6:8, 5] = bad[3, 6:8, 5] = True
    bad[0, 12:14] = bad[3, 12:14] = True
    bad[3, 1] = True
    bad[2, 0] = True
    assert torch.equal(out.view(4, 16, 128).isnan().cpu(), bad)
    want, mass = ref.attend(q.nan_to_num(nan=0.0, posinf=0.0), [0] * 4, pos)
    good = ~bad.view(4, -1)
    err = (out.double().cpu() - want).abs()
    assert (err <= 2.0 ** -8 * want.abs() + HALF * mass)[good].all()


# ---------------------------------------------------------------------------
# prefill
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,L", [(1, 2), (2, 3), (3, 4), (2, 5), (1, 8), (40, 6), (1, 12), (1, 13), (2, 21), (1, 160)])
def test_few_queries_over_long_contexts(n, L):
    """Contexts cut into many runs: against a binary64 product on the GPU."""
    pos0 = 6000 if n < 10 else 700
    c = fresh(2, pos0 + L, n_layers=1)
    for s in range(2):
        k, v = rows(pos0 + L, 1024, torch.float32, 250 + s).cuda(), rows(pos0 + L, 1024, torch.float32, 260 + s).cuda()
        n5.kv8_append(c, k, v, i32([s]), i32([0]), pos0 + L, 0)
    ids = [(s + 1) % 2 for s in range(n)]
    q = rows(n * L, 2048, torch.bfloat16, 270).cuda()
    out = n5.attention_prefill_kv8(q, c, i32(ids), L, pos0, 0)
    t = torch.arange(pos0 + L, device="cuda")
    for i, s in enumerate(ids[:4]):
        k = c.k[s, 0].double() * c.k_scale[s, 0][:, t // BLOCK, None].double()
        v = c.v[s, 0].double() * c.v_scale[s, 0][:, t // BLOCK, None].double()
        x = q[i * L:(i + 1) * L].double().view(L, 8, 2, 128).permute(1, 2, 0, 3).reshape(8, 2 * L, 128)
        w = (x @ k.transpose(1, 2) * 0.08838834764831845).view(8, 2, L, -1)
        w = torch.softmax(w.masked_fill(t > pos0 + torch.arange(L, device="cuda")[:, None], float("-inf")), -1)
        want, mass = ((w.view(8, 2 * L, -1) @ y).view(8, 2, L, 128).permute(2, 0, 1, 3).reshape(L, -1).cpu()
                      for y in (v, v.abs()))
        assert_near(out[i * L:(i + 1) * L], want, mass)


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("n,L,pos0", [
    (1, 1, 0), (3, 1, 131), (2, 2, 62), (3, 3, 126), (2, 4, 63), (2, 5, 0), (1, 8, 190), (2, 9, 100), (1, 16, 7),
    (2, 17, 50), (1, 33, 100), (2, 64, 0), (1, 130, 0), (1, 70, 61), (1, 131, 128), (1, 200, 60),
])
def test_prefill_matches_definition(n, L, pos0, workspace):
    lens = [pos0 + L, 3, pos0 + L, pos0 + L]
    c, ref = filled(4, pos0 + L + 11, 200 + L, lengths=lens)
    ids = [3, 0, 2][:n]
    q = rows(n * L, 2048, torch.bfloat16, 201)
    out = n5.attention_prefill_kv8(q.cuda(), c, i32(ids), L, pos0, 1, workspace=workspace)
    assert_near(out, *ref.attend(q, ids, [pos0] * n, L), weight=BF)
    assert n5.device_status() == n5.OK


def test_prefill_strides_and_bad_slots():
    c, ref = filled(2, 150, 230)
    for L in (3, 40):
        wide = rows(3 * L, 2304, torch.bfloat16, 231).cuda()
        buf = torch.full((3 * L + 2, 2176), 7.0, dtype=torch.bfloat16, device="cuda")
        n5.attention_prefill_kv8(wide, c, i32([1, 5, 0]), L, 77, 1, out=buf[:3 * L])
        want, mass = ref.attend(wide[:, :2048].cpu(), [1, 5, 0], [77] * 3, L)
        assert_near(buf[:3 * L, :2048], want, mass, BF)
        assert (buf[L:2 * L, :2048] == 0).all()
        assert (buf[:, 2048:] == 7).all() and (buf[3 * L:] == 7).all()


def test_prefill_rows_equal_decode():
    c, ref = filled(1, 400, 240)
    q = rows(150, 2048, torch.bfloat16, 241).cuda()
    pre = n5.attention_prefill_kv8(q, c, i32([0]), 150, 250, 1)
    at = [0, 1, 63, 64, 149]
    dec = n5.attention_decode_kv8(q[at].contiguous(), c, i32([0] * 5), i32([250 + i for i in at]), 1)
    _, mass = ref.attend(q[at].cpu(), [0] * 5, [250 + i for i in at])
    assert_near(pre[at], dec.double().cpu(), mass, BF + HALF + 2.0 ** -8)


# ---------------------------------------------------------------------------
# selection and sparse attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n_select,sink,recent", [(1, 0, 0), (1, 0, 1), (4, 1, 2), (5, 0, 0), (16, 3, 4), (40, 1, 1)])
@pytest.mark.parametrize("pos", [[0], [1499], [-1], [1499, 64, 63, 255, 256, 900, -1]])
def test_select_matches_definition(n_select, sink, recent, pos):
    n = len(pos)
    c, ref = filled(3, 1500, 300)
    ids = [(i + 1) % 3 for i in range(n)]
    q = rows(n, 2048, torch.bfloat16, 301)
    got = n5.kv8_select_blocks(q.cuda(), c, i32(ids), i32(pos), 1, n_select, sink, recent)
    assert torch.equal(got.cpu(), ref.select(q, ids, pos, n_select, sink, recent))


def test_select_ties_special_values_and_bad_slots():
    """Equal blocks: the lower index; a zero query ties them all; NaN queries rank nothing."""
    c = fresh(2, 64 * 20)
    k = rows(64, 1024, torch.float32, 310).repeat(20, 1)      # twenty equal blocks
    k[64 * 7:64 * 8] *= 4
    k[64 * 13:64 * 14] *= 4
    n5.kv8_append(c, k.cuda(), k.cuda(), i32([0]), i32([0]), 1280, 1)
    n5.kv8_append(c, k.cuda(), k.cuda(), i32([1]), i32([0]), 1280, 1)
    ref = Cache.of(c, 1)
    q = rows(5, 2048, torch.bfloat16, 311)
    q[1] = 0
    q[2] = float("nan")
    ids, pos = [0, 1, 0, 2, -3], [1279, 1279, 1279, 100, 100]
    for n_select, sink, recent in [(1, 0, 0), (6, 1, 1), (3, 0, 0)]:
        got = n5.kv8_select_blocks(q.cuda(), c, i32(ids), i32(pos), 1, n_select, sink, recent)
        assert torch.equal(got.cpu(), ref.select(q, ids, pos, n_select, sink, recent))
    assert (got[3:] == -1).all()


def test_select_many_blocks():
    """Over 4096 blocks, some in long runs of equal scores."""
    nb = 4500
    c = fresh(1, 64 * nb, n_layers=1)
    g = torch.Generator(device="cuda").manual_seed(5)
    kb = torch.randn((1, 1, 8, nb, 2, 128), device="cuda", generator=g)
    kb[:, :, :, 1000:1400] = kb[:, :, :, :1, :, :] + 0.3
    kb = kb.sort(dim=4).values
    c.k_bounds.copy_(kb.to(torch.float8_e4m3fn))
    c.k_scale.copy_(torch.exp2(torch.randint(-2, 2, c.k_scale.shape, device="cuda", generator=g).float()))
    ref = Cache.of(c, 0)
    q = rows(1, 2048, torch.bfloat16, 312, 3.0)
    for n_select in (1, 64, 1500, 4499, 5000):
        got = n5.kv8_select_blocks(q.cuda(), c, i32([0]), i32([64 * nb - 30]), 0, n_select, 1, 0)
        lo, hi = kb_values(ref, nb)
        qq = q.double().view(8, 2, 1, 128)
        score = torch.maximum(qq * lo, qq * hi).sum(-1).amax(1) * ref.scale["k"][0]
        score[:, 0] = float("inf")
        order = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :n_select].sort(-1).values
        want = torch.full((8, n_select), -1, dtype=torch.int64)
        want[:, :order.shape[1]] = order
        assert torch.equal(got[0].cpu().long(), want), n_select


def kb_values(ref, nb):
    from kv8_oracle import values
    v = values(ref.bounds[0])                                  # [8, nb, 2, 128]
    return v[:, None, :, 0], v[:, None, :, 1]


@pytest.mark.parametrize("split", [True, False])
def test_sparse_matches_definition(split):
    c, ref = filled(3, 700, 320)
    ids, pos = [2, 0, 1, 1, 0], [699, 64, 130, -1, 320]
    q = rows(5, 2048, torch.bfloat16, 321)
    blocks = torch.full((5, 8, 6), -1, dtype=torch.int32)
    g = gen(7)
    for s in range(5):
        for h in range(8):
            n = int(torch.randint(0, 7, (1,), generator=g))
            # any order, past the context too, holes between
            blocks[s, h, torch.randperm(6, generator=g)[:n]] = torch.randperm(12, generator=g)[:n].to(torch.int32)
    blocks[0, 0] = torch.tensor([3, 3, 0, -7, 2147483647, -2147483648], dtype=torch.int32)   # twice, and nonsense
    blocks[0, 1] = -1                                                                        # nothing
    blocks[1, 2] = torch.tensor([1, -1, -1, -1, -1, -1], dtype=torch.int32)                  # one position
    out = n5.attention_sparse_kv8(q.cuda(), c, i32(ids), i32(pos), blocks.cuda(), 1, split=split)
    sane = blocks.clone()
    sane[blocks > 11] = -1
    want, mass = ref.attend(q, ids, pos, blocks=sane.tolist())
    assert_near(out, want, mass)
    assert (out[0, 256:512] == 0).all() and (out[3] == 0).all()
    empty = n5.attention_sparse_kv8(q.cuda(), c, i32(ids), i32(pos), blocks[:, :, :0].contiguous().cuda(), 1,
                                    split=split)
    assert (empty == 0).all()


@pytest.mark.parametrize("split", [True, False])
def test_sparse_long_lists_with_holes(split):
    """Lists of several batches of 32 entries, with whole batches of nothing."""
    c, ref = filled(2, 2000, 340)
    ids, pos = [1, 0, 1], [1999, 1200, 100]
    q = rows(3, 2048, torch.bfloat16, 341)
    n_select = 150
    g = gen(9)
    blocks = torch.full((3, 8, n_select), -1, dtype=torch.int32)
    for s in range(3):
        for h in range(8):
            at = torch.randperm(n_select, generator=g)[:[0, 1, 3, 20, 32, 32, 5, 12][h]]
            if h == 4:
                at = torch.arange(118, 150)                      # the last batches alone
            if h == 5:
                at = torch.arange(0, 32)                         # the first alone
            if h == 6:
                at = torch.tensor([31, 32, 63, 64, 149])
            blocks[s, h, at] = torch.randperm(32, generator=g)[:at.numel()].to(torch.int32)
    out = n5.attention_sparse_kv8(q.cuda(), c, i32(ids), i32(pos), blocks.cuda(), 1, split=split)
    assert_near(out, *ref.attend(q, ids, pos, blocks=blocks.tolist()))
    assert n5.device_status() == n5.OK


def test_sparse_over_all_blocks_is_decode():
    c, ref = filled(2, 1000, 330)
    ids, pos = [1, 0, 1], [999, 500, 63]
    q = rows(3, 2048, torch.bfloat16, 331)
    blocks = n5.kv8_select_blocks(q.cuda(), c, i32(ids), i32(pos), 1, 16, 1, 2)
    out = n5.attention_sparse_kv8(q.cuda(), c, i32(ids), i32(pos), blocks, 1)
    assert_near(out, *ref.attend(q, ids, pos))


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_prompt_then_tokens_with_selection():
    """A prompt appended in two chunks with its attention, then tokens appended and
    decoded, dense and over selected blocks, as a program serves them."""
    ids, n, max_len = [2, 0], 2, 400
    c, ref = fresh(3, max_len), Cache.of(fresh(3, max_len), 1)
    sid = i32(ids)
    at = 0
    for L in (150, 101):
        k, v, q = (rows(n * L, w, torch.bfloat16, at + i) for i, w in enumerate((1024, 1024, 2048)))
        pos = i32([at] * n)
        n5.kv8_append(c, k.cuda(), v.cuda(), sid, pos, L, 1)
        ref.append(k, v, ids, [at] * n, L)
        out = n5.attention_prefill_kv8(q.cuda(), c, sid, L, at, 1)
        assert_near(out, *ref.attend(q, ids, [at] * n, L), weight=BF)
        at += L
    pos = i32([at] * n)
    for step in range(12):
        k, v, q = (rows(n, w, torch.float32, 900 + 3 * step + i, 1 + step) for i, w in enumerate((1024, 1024, 2048)))
        q = q.to(torch.bfloat16)
        n5.kv8_append(c, k.cuda(), v.cuda(), sid, pos, 1, 1)
        ref.append(k, v, ids, [at] * n, 1)
        dense = n5.attention_decode_kv8(q.cuda(), c, sid, pos, 1)
        assert_near(dense, *ref.attend(q, ids, [at] * n), weight=HALF + 2.0 ** -9)
        blocks = n5.kv8_select_blocks(q.cuda(), c, sid, pos, 1, 3, 1, 1)
        assert torch.equal(blocks.cpu(), ref.select(q, ids, [at] * n, 3, 1, 1))
        out = n5.attention_sparse_kv8(q.cuda(), c, sid, pos, blocks, 1)
        assert_near(out, *ref.attend(q, ids, [at] * n, blocks=blocks.cpu().tolist()), weight=HALF + 2.0 ** -9)
        pos += 1
        at += 1
    assert_state(c, ref, 1)


def test_workspaces_of_the_c_interface():
    """Garbage in the workspace changes nothing; one too small or unaligned counts as none."""
    import ctypes as C
    L = n5.lib()
    c, ref = filled(2, 3000, 430)
    q, ids, pos = rows(2, 2048, torch.bfloat16, 431).cuda(), i32([1, 0]), i32([2999, 2000])
    st = torch.cuda.current_stream().cuda_stream
    need = L.n550_attention_kv8_workspace(2)
    ws = torch.empty(need + 32, dtype=torch.uint8, device="cuda")

    def call(ptr, n):
        out = torch.empty((2, 2048), dtype=torch.bfloat16, device="cuda")
        assert L.n550_attention_decode_kv8(st, q.data_ptr(), 2048, C.byref(c._c), 1, ids.data_ptr(), pos.data_ptr(), 2,
                                           out.data_ptr(), 2048, ptr, n) == n5.OK
        return out

    got = []
    for fill in (0, 0x7F, 0xFF):
        ws.fill_(fill)
        got.append(call(ws.data_ptr(), need))
    assert_near(got[0], *ref.attend(q.cpu(), [1, 0], [2999, 2000]))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    whole = call(None, 0)
    for ptr, n in ((ws.data_ptr(), need - 1), (ws.data_ptr() + 8, need)):
        assert torch.equal(call(ptr, n), whole)
    q40 = rows(2 * 40, 2048, torch.bfloat16, 432).cuda()
    out = torch.empty((80, 2048), dtype=torch.bfloat16, device="cuda")
    assert L.n550_attention_prefill_kv8(st, q40.data_ptr(), 2048, C.byref(c._c), 1, ids.data_ptr(), 2, 40, 100,
                                        out.data_ptr(), 2048, ws.data_ptr(), 64) == n5.OK
    assert torch.equal(out, n5.attention_prefill_kv8(q40, c, ids, 40, 100, 1, workspace=False))


def test_captured_step_replays_on_new_inputs():
    """append + select + sparse + decode + prefill in one CUDA graph on a side stream,
    replayed with other inputs and positions in the same buffers."""
    n, max_len = 3, 520
    c, ref = filled(3, max_len, 400, lengths=[500, 400, 300])
    sid, pos = i32([0, 1, 2]), i32([500, 400, 300])
    k, v, q = (torch.empty((n, w), dtype=torch.bfloat16, device="cuda") for w in (1024, 1024, 2048))
    outs = [torch.empty((n, 2048), dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    blocks = torch.empty((n, 8, 3), dtype=torch.int32, device="cuda")

    def step():
        n5.kv8_append(c, k, v, sid, pos, 1, 1)
        n5.kv8_select_blocks(q, c, sid, pos, 1, 3, 1, 1, out=blocks)
        n5.attention_sparse_kv8(q, c, sid, pos, blocks, 1, out=outs[0])
        n5.attention_decode_kv8(q, c, sid, pos, 1, out=outs[1])
        n5.attention_prefill_kv8(q, c, sid, 1, 290, 1, out=outs[2])

    def feed(i):
        new = [rows(n, w, torch.bfloat16, 410 + 3 * i + j, 1.0 + i) for j, w in enumerate((1024, 1024, 2048))]
        for dst, src in zip((k, v, q), new):
            dst.copy_(src)
        return new

    def check(new, p):
        ids = [0, 1, 2]
        ref.append(new[0], new[1], ids, p, 1)
        assert_state(c, ref, 1)
        w = HALF + 2.0 ** -9
        assert torch.equal(blocks.cpu(), ref.select(new[2], ids, p, 3, 1, 1))
        assert_near(outs[0], *ref.attend(new[2], ids, p, blocks=blocks.cpu().tolist()), weight=w)
        assert_near(outs[1], *ref.attend(new[2], ids, p), weight=w)
        assert_near(outs[2], *ref.attend(new[2], ids, [290] * 3), weight=BF + 2.0 ** -9)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        new = feed(0)
        step()
    side.synchronize()
    check(new, [500, 400, 300])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in (1, 2, 3):
        new = feed(i)
        pos += 1
        graph.replay()
        torch.cuda.synchronize()
        check(new, [500 + i, 400 + i, 300 + i])


def test_two_streams_at_once():
    c, ref = filled(4, 3000, 500, lengths=[3000, 2000, 100, 2999])
    q = [rows(2, 2048, torch.bfloat16, 501 + i) for i in range(2)]
    dev = [x.cuda() for x in q]
    ids, pos = [[0, 1], [3, 2]], [[2999, 1999], [2998, 99]]
    args = [(i32(ids[i]), i32(pos[i])) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(n5.attention_decode_kv8(dev[i], c, *args[i], 1))
    torch.cuda.synchronize()
    for i in range(2):
        assert_near(got[i][0], *ref.attend(q[i], ids[i], pos[i]))
        for g in got[i][1:]:
            assert torch.equal(g, got[i][0])                 # the same bits every time


def test_cache_beyond_32_bit_offsets():
    """Slots and positions whose byte offsets pass 2^32."""
    max_len = 1_500_000
    c = n5.KV8Cache(4, max_len, n_layers=1)                   # 6.1 GB each of K and V
    p0 = max_len - 130
    for s, p in ((3, 0), (3, p0)):
        k, v = rows(130, 1024, torch.float32, 600 + p % 7).cuda(), rows(130, 1024, torch.float32, 610 + p % 7).cuda()
        n5.kv8_append(c, k, v, i32([s]), i32([p]), 130, 0)
    q = rows(1, 2048, torch.bfloat16, 620).cuda()
    last = (max_len - 1) // BLOCK
    blocks = torch.tensor([[[0, 1, last - 1, last]] * 8], dtype=torch.int32, device="cuda")
    out = n5.attention_sparse_kv8(q, c, i32([3]), i32([max_len - 1]), blocks, 0)
    t = torch.cat([torch.arange(128), torch.arange((last - 1) * BLOCK, max_len)]).cuda()
    k = c.k[3, 0].view(torch.uint8)[:, t].view(torch.float8_e4m3fn).double() * c.k_scale[3, 0][:, t // BLOCK, None].double()
    v = c.v[3, 0].view(torch.uint8)[:, t].view(torch.float8_e4m3fn).double() * c.v_scale[3, 0][:, t // BLOCK, None].double()
    w = torch.softmax(q[0].double().view(8, 2, 128) @ k.transpose(1, 2) * 0.08838834764831845, -1)
    assert_near(out[0], (w @ v).view(-1).cpu(), (w @ v.abs()).view(-1).cpu())
    short = n5.attention_decode_kv8(q, c, i32([3]), i32([129]), 0)
    pre = n5.attention_prefill_kv8(q, c, i32([3]), 1, 129, 0)
    k = c.k[3, 0, :, :130].double() * c.k_scale[3, 0][:, torch.arange(130, device="cuda") // BLOCK, None].double()
    v = c.v[3, 0, :, :130].double() * c.v_scale[3, 0][:, torch.arange(130, device="cuda") // BLOCK, None].double()
    w = torch.softmax(q[0].double().view(8, 2, 128) @ k.transpose(1, 2) * 0.08838834764831845, -1)
    for got in (short, pre):
        assert_near(got[0], (w @ v).view(-1).cpu(), (w @ v.abs()).view(-1).cpu(), BF)


def test_wrapper_refusals():
    c, _ = filled(2, 100, 700)
    q, sid, pos = rows(2, 2048, torch.bfloat16, 701).cuda(), i32([0, 1]), i32([99, 5])
    with pytest.raises(ValueError):
        n5.attention_decode_kv8(q.float(), c, sid, pos, 1)
    with pytest.raises(ValueError):
        n5.attention_decode_kv8(q[:1], c, sid, pos, 1)
    with pytest.raises(ValueError):
        n5.attention_decode_kv8(q, c, sid.long(), pos, 1)
    with pytest.raises(ValueError):
        n5.attention_decode_kv8(q, c, sid, pos[:1], 1)
    with pytest.raises(ValueError):
        n5.attention_decode_kv8(q, c, sid, pos.cpu(), 1)
    with pytest.raises(n5.N550Error):
        n5.attention_decode_kv8(q, c, sid, pos, 2)            # layer
    with pytest.raises(n5.N550Error):
        n5.attention_prefill_kv8(q, c, sid, 1, 100, 1)        # past the cache
    with pytest.raises(ValueError):
        n5.attention_sparse_kv8(q, c, sid, pos, torch.zeros((2, 4, 3), dtype=torch.int32, device="cuda"), 1)
    with pytest.raises(n5.N550Error):
        n5.kv8_select_blocks(q, c, sid, pos, 1, 2, 2, 1)
    with pytest.raises(ValueError):
        n5.kv8_append(c, q[:, :1024], q[:, :1024].float(), sid, pos, 1, 1)
    off = torch.empty(2 * 2048 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(2, 2048)
    with pytest.raises(n5.N550Error):
        n5.attention_decode_kv8(off, c, sid, pos, 1)          # not 16-byte aligned


@pytest.mark.parametrize("fill", [0x00, 0x7F, 0xFF, None])
def test_merge_skips_records_that_no_run_wrote(fill):
    """The merge after an attention kernel that gave up before its records were written:
    whatever the workspace holds, only rows of records that name a pair and pieces of the
    call are written. (1 << 30 pieces, a sequence or a head that is not there and one
    piece too many would otherwise lead out of the workspace and out of `out`.)"""
    L, n, runs = n5.lib(), 3, 444                             # 148 SMs x 3 CTAs
    need = L.n550_attention_kv8_workspace(n)
    assert need == runs * (16 + 2 * 2 * 130 * 4)
    ws = torch.zeros(need // 4, dtype=torch.int32, device="cuda")
    rec = ws[:4 * runs].view(runs, 4)                         # sequence, KV head, pieces, slot
    part = ws[4 * runs:].view(torch.float32).view(2 * runs, 2 * 130)
    big = 2147483647
    if fill is not None:
        ws.view(torch.uint8).fill_(fill)
    else:
        rec[:, :] = torch.tensor([[0, 0, 1 << 30, 0], [n, 0, 2, 0], [-1, 0, 2, 0], [0, 8, 2, 0], [0, -1, 2, 0], [0, 0, -1, 0],
                                  [0, 0, -big - 1, 0], [big, 0, 2, 0], [0, big, 2, 0], [0, 0, runs - 8, 0], [0, 0, big, 0],
                                  [0, 0, 0, 0]], dtype=torch.int32).repeat(37, 1).cuda()
        for c in range(9, runs, 12):
            rec[c, 2] = runs - c + 1                          # one piece more than there are runs
    out = torch.full((n + 2, 2048), 7.0, dtype=torch.bfloat16, device="cuda")
    rows_ = out[1:1 + n]

    def merge():
        n5.check(L.n550_check_kv8_merge(n5.stream_ptr(), n, ws.data_ptr(), need, rows_.data_ptr(), 2048))
        torch.cuda.synchronize()

    merge()
    assert (out == 7).all()
    # one record among them that a run wrote: pieces in runs 440 and 441, the first in slot 881
    rec[440] = i32([2, 5, 2, 881])
    part[881, :256], part[881, 256:] = 3.0, torch.tensor([1.0, 4.0, 1.0, 4.0], device="cuda")
    part[882, :256], part[882, 256:] = 5.0, torch.tensor([1.0, 4.0, 1.0, 4.0], device="cuda")
    merge()
    want = torch.full((n + 2, 2048), 7.0, dtype=torch.bfloat16)
    want[3, 5 * 256:6 * 256] = 1.0                            # (3 + 5) / (4 + 4)
    assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("pos0", [1, 1 << 30, 2 ** 31 - 1])
def test_prefill_past_the_cache_is_refused_before_its_workspace(pos0):
    """The workspace of 300 queries at 2^30 would be 4 TB: the call is refused as such."""
    c, _ = filled(1, 300, 720)
    with pytest.raises(n5.N550Error) as e:
        n5.attention_prefill_kv8(rows(300, 2048, torch.bfloat16, 721).cuda(), c, i32([0]), 300, pos0, 1)
    assert e.value.status == n5.ERR_ARG


@pytest.mark.parametrize("qmax,kmax", [(2.0 ** 127.5, 2.0 ** -121), (2.0 ** 125, 2.0 ** -119), (2.0 ** -121, 2.0 ** 127), (2.0 ** -119, 2.0 ** 125)])
@pytest.mark.parametrize("L", [1, 3, 7])
def test_scores_of_queries_and_keys_at_the_ends_of_the_range(qmax, kmax, L):
    """Queries near BF16's largest number over keys near its smallest, and the other way
    round: their products are ordinary numbers, and so are the scores.

    A score is a sum of 128 products of at most qmax kmax = 2^6.5, so below 2^13.5 before
    the factor 2^-3.5: 128 roundings of partial sums that are below 2^13.5 move it by at
    most 128 * 2^-24 * 2^13.5 * 2^-3.5 = 2^-7 (and a weight by that part of it). A query's
    smallest parts are 2^-21 of its largest, half of which in 128 products with keys is
    128 * 2^-22 * 2^6.5 * 2^-3.5 = 2^-12 more; the keys, of 4 bits, are what the cache
    holds, also where their scale is 2^-126."""
    n = 150
    c = fresh(2, n)
    g = gen(730)
    k = (torch.rand((n, 1024), generator=g) * 2 - 1) * kmax
    v = rows(n, 1024, torch.float32, 731)
    n5.kv8_append(c, k.cuda(), v.cuda(), i32([1]), i32([0]), n, 1)
    ref = Cache.of(c, 1)
    q = ((torch.rand((L, 2048), generator=g) * 2 - 1) * qmax).to(torch.bfloat16)
    out = n5.attention_prefill_kv8(q.cuda(), c, i32([1]), L, n - L, 1)
    assert_near(out, *ref.attend(q, [1], [n - L], L), weight=HALF + 2.0 ** -7 + 2.0 ** -11)
    if L == 1:
        for split in (True, False):
            out = n5.attention_decode_kv8(q.cuda(), c, i32([1]), i32([n - 1]), 1, split=split)
            assert_near(out, *ref.attend(q, [1], [n - 1]), weight=HALF + 2.0 ** -7 + 2.0 ** -11)


def prefill_with(c, q, ids, L, pos0, nbytes):
    """n550_attention_prefill_kv8 with a workspace of nbytes, nothing behind which is written."""
    import ctypes as C
    ws = torch.full((nbytes + 4096,), 0x7F, dtype=torch.uint8, device="cuda")
    out = torch.empty((len(ids) * L, 2048), dtype=torch.bfloat16, device="cuda")
    n5.check(n5.lib().n550_attention_prefill_kv8(n5.stream_ptr(), q.data_ptr(), 2048, C.byref(c._c), 1, i32(ids).data_ptr(), len(ids),
                                                 L, pos0, out.data_ptr(), 2048, ws.data_ptr() if nbytes else None, nbytes))
    torch.cuda.synchronize()
    assert (ws[nbytes:] == 0x7F).all()
    return out


def test_prefill_in_groups_of_what_the_workspace_holds():
    """A workspace of some of the sequences: the same bits as with all of them (one
    sequence's rows do not depend on the others); of less than one, passes."""
    L, pos0 = 130, 70
    c, ref = filled(3, pos0 + L, 740)
    ids = [2, 0, 5, 1, 0, 2, 1]                               # (a slot that is not there, too)
    q = rows(len(ids) * L, 2048, torch.bfloat16, 741).cuda()
    one = 4096 * (pos0 + L)
    assert n5.lib().n550_attention_prefill_kv8_workspace(len(ids), L, pos0) == len(ids) * one
    want = prefill_with(c, q, ids, L, pos0, len(ids) * one)
    assert_near(want, *ref.attend(q.cpu(), ids, [pos0] * len(ids), L), weight=BF)
    for nbytes in (one, 2 * one, 3 * one + 100, 4 * one, 6 * one, 7 * one - 1, 9 * one):
        assert torch.equal(prefill_with(c, q, ids, L, pos0, nbytes), want), nbytes
    none = prefill_with(c, q, ids, L, pos0, 0)
    assert torch.equal(prefill_with(c, q, ids, L, pos0, one - 1), none)
    assert_near(none, *ref.attend(q.cpu(), ids, [pos0] * len(ids), L))
    assert n5.device_status() == n5.OK


def test_prefill_splits_with_a_workspace_too_small_for_a_sequence():
    """Room for the splits' partials, but for no context as BF16."""
    L, pos0, ids = 20, 1900, [1, 0, 1, 0, 1, 0, 1, 0, 1, 0, 1, 0]
    c, _ = filled(2, pos0 + L, 750)
    q = rows(len(ids) * L, 2048, torch.bfloat16, 751).cuda()
    lb = n5.lib()
    split, one = lb.n550_attention_prefill_kv8_workspace(len(ids), 8, pos0), 4096 * (pos0 + L)
    assert split < one < lb.n550_attention_prefill_kv8_workspace(len(ids), L, pos0)
    got = prefill_with(c, q, ids, L, pos0, split)
    # passes of 8, 8 and 4 queries with splits
    for j in (0, 8, 16):
        m = min(8, L - j)
        part = q.view(len(ids), L, 2048)[:, j:j + m].reshape(-1, 2048).contiguous()
        want = n5.attention_prefill_kv8(part, c, i32(ids), m, pos0 + j, 1)
        assert torch.equal(got.view(len(ids), L, 2048)[:, j:j + m], want.view(len(ids), m, 2048))
    # and without: as with no workspace at all
    assert torch.equal(prefill_with(c, q, ids, L, pos0, split - 1), prefill_with(c, q, ids, L, pos0, 0))


def test_prefill_wrapper_caps_its_workspace(monkeypatch):
    c, _ = filled(2, 400, 760)
    ids = i32([1, 0, 1, 0, 0])
    q = rows(5 * 200, 2048, torch.bfloat16, 761).cuda()
    want = n5.attention_prefill_kv8(q, c, ids, 200, 200, 1)
    most = []
    was = n5.kv8._workspace
    monkeypatch.setattr(n5.kv8, "_workspace", lambda nbytes, q: most.append(nbytes) or was(nbytes, q))
    for cap, nbytes in ((5 * 400 * 4096, 5 * 400 * 4096), (2 * 400 * 4096 + 7, 2 * 400 * 4096 + 7), (1, 400 * 4096)):
        monkeypatch.setattr(n5.kv8, "PREFILL_WORKSPACE_MAX", cap)
        assert torch.equal(n5.attention_prefill_kv8(q, c, ids, 200, 200, 1), want)
        assert most.pop() == nbytes


@pytest.mark.parametrize("e", [-124, -60, 0, 119])
def test_attention_reads_values_at_the_ends_of_the_range(e):
    """One position's V is what every code times 2^e is, to the bit, on both prefill
    routes and in decode; the others' are zero, and so are the scores."""
    n = 140
    v0 = torch.arange(128, dtype=torch.uint8).view(torch.float8_e4m3fn).float().nan_to_num(nan=448.0)
    v0[1::2] *= -1
    v = torch.zeros((n, 8, 128))
    v[0] = v0 * 2.0 ** e
    c = fresh(1, n)
    n5.kv8_append(c, torch.zeros((n, 1024), device="cuda"), v.view(n, 1024).cuda(), i32([0]), i32([0]), n, 1)
    assert (c.v_scale[0, 1, :, 0] == 2.0 ** e).all()
    q = rows(n, 2048, torch.bfloat16, 770).cuda()
    want = v[0].to(torch.bfloat16)[:, None].expand(8, 2, 128)
    for out in (n5.attention_decode_kv8(q[:1], c, i32([0]), i32([0]), 1), n5.attention_prefill_kv8(q[:5], c, i32([0]), 5, 0, 1),
                n5.attention_prefill_kv8(q, c, i32([0]), n, 0, 1)):
        assert torch.isfinite(out).all()
        assert torch.equal(out[0].view(8, 2, 128).cpu().float(), want.float())


def test_the_tensors_of_a_cache_stay_its_tensors():
    """The library holds their addresses: an assignment would leave the calls with the old
    tensor's memory, freed or not."""
    c = n5.KV8Cache(1, 64, n_layers=1)
    for name in ("k", "v", "k_scale", "v_scale", "k_bounds"):
        t = getattr(c, name)
        with pytest.raises(AttributeError):
            setattr(c, name, t.clone())
        assert getattr(c, name) is t
    assert (c._c.k, c._c.v, c._c.k_scale, c._c.v_scale, c._c.k_bounds) == tuple(
        t.data_ptr() for t in (c.k, c.v, c.k_scale, c.v_scale, c.k_bounds))
    assert n5.KV8Cache(1, 64, n_layers=1, bounds=False).k_bounds is None


@pytest.mark.parametrize("strange", [float("nan"), float("inf"), -float("inf")])
def test_select_with_one_strange_head(strange):
    """A NaN in one of a KV head's two query heads leaves the other's order; an infinity
    puts every block with that sign of K in the channel first (lower index among equals)."""
    c, ref = filled(2, 1000, 780)
    q = rows(3, 2048, torch.bfloat16, 781)
    q[0, 5 * 128 + 7] = strange
    q[2, 12 * 128] = strange
    ids, pos = [1, 0, 1], [999, 700, 640]
    for n_select, sink, recent in [(4, 1, 1), (7, 0, 0)]:
        got = n5.kv8_select_blocks(q.cuda(), c, i32(ids), i32(pos), 1, n_select, sink, recent)
        assert torch.equal(got.cpu(), ref.select(q, ids, pos, n_select, sink, recent))
