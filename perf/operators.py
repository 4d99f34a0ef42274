"""The operators of the 8-bit KV cache: what is timed, and their plain forms.

The cache holds K and V of 8 KV heads x 128 dimensions as e4m3 codes, with one
power-of-two scale for each block of 64 positions and KV head, and for each
block and K channel the smallest and the largest code (the block's bounds).

  append   quantise n x L new K/V rows into the cache behind what it holds
  decode   one query per sequence over its whole context
  prefill  L queries per sequence, causal, over a context that ends with them
  select   the blocks whose bounds promise the largest scores for a query
  sparse   one query per sequence over the selected blocks alone

`run` computes them in plain torch operations (own = False) or through the
framework's entry points (own = True) on the state `prepare` makes.
"""
import math

import torch

own = False

DEV = "cuda"
HEADS, KVH, HD, BLOCK = 16, 8, 128, 64
SCALE = 0.08838834764831845
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a decode step of the batched benchmark: 256 sequences, one FP32 row each
        dict(name="append_256x1", op="append", n=256, L=1, ctx=1024, ragged=True, f32=True),
        # the K/V rows of a 64 x 512-token prompt batch
        dict(name="append_64x512", op="append", n=64, L=512, ctx=0, ragged=False, f32=False),
        # one interactive user at a short context: latency
        dict(name="decode_1x1152", op="decode", n=1, ctx=1152, ragged=False),
        # a decode step of the batched benchmark
        dict(name="decode_256x1152", op="decode", n=256, ctx=1152, ragged=True),
        # a few long documents of very different lengths
        dict(name="decode_4x131072", op="decode", n=4, ctx=131072, ragged=True),
        # the prompt batch of the prefill benchmark
        dict(name="prefill_64x512", op="prefill", n=64, L=512, pos0=0),
        # a later chunk of two long prompts, off the block grid
        dict(name="prefill_2x2048", op="prefill", n=2, L=2048, pos0=4100),
        # verification of four drafted tokens for eight users
        dict(name="verify_8x5", op="prefill", n=8, L=5, pos0=2043),
        # block selection for one very long context, and for a batch of long ones
        dict(name="select_1x131072", op="select", n=1, ctx=131072, ragged=False, blocks=64, sink=1, recent=2),
        dict(name="select_16x32768", op="select", n=16, ctx=32768, ragged=True, blocks=32, sink=1, recent=2),
        # and the attention over what was selected
        dict(name="sparse_1x131072", op="sparse", n=1, ctx=131072, ragged=False, blocks=64),
        dict(name="sparse_16x32768", op="sparse", n=16, ctx=32768, ragged=True, blocks=32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill", "select", "sparse"])
    if op == "append":
        L = rng.choice([1, 1, _log(rng, 2, 512)])
        n = _log(rng, 1, max(1, min(256, 32768 // L)))
        return dict(op=op, n=n, L=L, ctx=_log(rng, 1, 2000) if rng.random() < 0.7 else 0,
                    ragged=rng.random() < 0.7, f32=rng.random() < 0.5)
    if op == "prefill":
        L = _log(rng, 2, 2048)
        n = _log(rng, 1, max(1, min(64, 4096 // L)))
        return dict(op=op, n=n, L=L, pos0=0 if rng.random() < 0.3 else _log(rng, 1, 4100))
    ctx = _log(rng, 4096 if op == "select" else 1, 131072)        # select: more blocks than it takes
    n = _log(rng, 1, max(1, min(256, 250000 // ctx)))
    case = dict(op=op, n=n, ctx=ctx, ragged=rng.random() < 0.7)
    if op != "decode":
        case["blocks"] = _log(rng, 4, min(96, max(4, ctx // (2 * BLOCK))))
    if op == "select":
        case["sink"], case["recent"] = rng.randint(0, 2), rng.randint(1, 2)
    return case


def _lengths(case):
    """Positions that each sequence's query attends to (append: that its slot holds before)."""
    n, ctx = case["n"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * n
    if n <= 32:
        return [max(min(ctx, 1), ctx // (1 + 3 * (i % 4)) - 5 * i) for i in range(n)]
    return [max(min(ctx, 1), ctx - 7 * (i % 37)) for i in range(n)]


def _nb(t):
    return -(-t // BLOCK)


def work(case):
    n, op = case["n"], case["op"]
    if op == "append":
        L, esz = case["L"], 4 if case["f32"] else 2
        blocks = sum(_nb(t + L) - t // BLOCK for t in _lengths(case))
        old = sum(1 for t in _lengths(case) if t % BLOCK)
        rows = n * L * KVH * HD
        # rows in, codes out, scales and bounds of the touched blocks out (in too where the block held tokens)
        return dict(bytes=rows * 2 * (esz + 1) + (blocks + old) * KVH * (2 * HD + 8) + 8 * n, flops=rows * 2 * 4)
    if op == "prefill":
        L, pos0 = case["L"], case["pos0"]
        t = pos0 + L
        pairs = n * sum(range(pos0 + 1, t + 1))
        return dict(bytes=n * KVH * (t * 2 * HD + _nb(t) * 8) + n * L * HEADS * HD * 4 + 4 * n,
                    flops=pairs * HEADS * HD * 4)
    lens = _lengths(case)
    io = n * HEADS * HD * 4 + 8 * n
    if op == "decode":
        return dict(bytes=io + sum(KVH * (t * 2 * HD + _nb(t) * 8) for t in lens),
                    flops=sum(lens) * HEADS * HD * 4)
    if op == "select":
        blocks = sum(_nb(t) for t in lens)
        return dict(bytes=io - n * HEADS * HD * 2 + blocks * KVH * (2 * HD + 4) + n * KVH * case["blocks"] * 4,
                    flops=blocks * HEADS * HD * 4)
    tokens = sum(min(t, case["blocks"] * BLOCK - (BLOCK - 1 - (t - 1) % BLOCK)) for t in lens)
    blocks = sum(min(_nb(t), case["blocks"]) for t in lens)
    return dict(bytes=io + KVH * (tokens * 2 * HD + blocks * 12), flops=tokens * HEADS * HD * 4)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s (FP32; 2^-126 for 0)."""
    m, e = torch.frexp(amax)
    s = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    s = torch.where(amax > 0, s, torch.full_like(s, -126))
    return torch.exp2(s.double()).float()


def _codes(x, scale):
    return (x / scale).clamp(-448.0, 448.0).to(E4M3)


def _filled(gen, slots, max_len, chan):
    """Codes, scales and bounds of a cache whose slots hold max_len positions."""
    nb = _nb(max_len)
    x = torch.randn((slots, 1, KVH, nb * BLOCK, HD), device=DEV, generator=gen)
    x *= torch.exp(0.3 * torch.randn((slots, 1, KVH, nb * BLOCK, 1), device=DEV, generator=gen)) * chan
    x = x.view(slots, 1, KVH, nb, BLOCK, HD)
    scale = _scale_of(x.abs().amax((-1, -2)))
    c = _codes(x, scale[..., None, None])
    f = c.to(torch.float16)
    bounds = torch.stack([f.amin(-2), f.amax(-2)], dim=-2).to(E4M3)
    c = c.view(slots, 1, KVH, nb * BLOCK, HD)[:, :, :, :max_len]
    return c.contiguous(), scale, bounds


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, n = case["op"], case["n"]
    L = case.get("L", 1)
    if op == "prefill":
        before = [case["pos0"]] * n
    elif op == "append":
        before = _lengths(case)
    else:
        before = [t - 1 for t in _lengths(case)]
    max_len = max(before) + L
    if op != "prefill":
        max_len += 5                      # room behind the last sequence's end
    chan = torch.exp(0.5 * torch.randn((1, 1, KVH, 1, HD), device=DEV, generator=gen))
    k, k_scale, k_bounds = _filled(gen, n + 1, max_len, chan)
    v, v_scale, _ = _filled(gen, n + 1, max_len, 1.0)
    order = torch.randperm(n, device=DEV, generator=gen)
    state = dict(case=dict(case), L=L, k=k, v=v, k_scale=k_scale, v_scale=v_scale, k_bounds=k_bounds,
                 seq_ids=torch.randperm(n + 1, device=DEV, generator=gen)[:n].to(torch.int32),
                 pos=torch.tensor(before, dtype=torch.int32, device=DEV)[order].contiguous())
    if op == "append":
        dt = torch.float32 if case["f32"] else torch.bfloat16
        k_new = torch.randn((n * L, KVH, HD), device=DEV, generator=gen) * chan.view(1, KVH, HD)
        state["k_new"] = k_new.to(dt).view(n * L, KVH * HD)
        state["v_new"] = torch.randn((n * L, KVH * HD), device=DEV, generator=gen).to(dt)
    else:
        q = torch.randn((n * L, KVH, 2, HD), device=DEV, generator=gen) / chan.view(1, KVH, 1, HD).clamp(min=0.5)
        state["q"] = (1.5 * q).to(torch.bfloat16).view(n * L, HEADS * HD)
    if op == "sparse":
        nb = state["pos"].long() // BLOCK + 1
        width = _nb(max_len)
        score = torch.rand((n, KVH, width), device=DEV, generator=gen)
        idx = torch.arange(width, device=DEV)
        score = torch.where(idx == nb[:, None, None] - 1, 2.0, score)
        state["blocks"] = _first_blocks(score.double(), nb, case["blocks"])
    if own:                               # the handle a program keeps beside its cache
        import n550_qwen3_bringup_handover_b200 as n5
        state["cache"] = n5.KV8Cache(k=k, v=v, k_scale=k_scale, v_scale=v_scale, k_bounds=k_bounds)
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _first_blocks(score, nb, n_select):
    """Indices of the n_select largest scores among the first nb blocks, ascending, -1 behind the last."""
    width = score.shape[-1]
    idx = torch.arange(width, device=score.device)
    score = torch.where(idx < nb[:, None, None], score, float("-inf"))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :n_select]
    rank = torch.arange(order.shape[-1], device=score.device)
    order = torch.where(rank < nb[:, None, None], order, width)
    order = torch.sort(order, dim=-1).values
    order = torch.where(order < width, order, -1)
    if order.shape[-1] < n_select:
        order = torch.nn.functional.pad(order, (0, n_select - order.shape[-1]), value=-1)
    return order.to(torch.int32).contiguous()


def _values(codes, scale, slots):
    """FP32 values [n, KVH, T, HD] of the slots of a cache."""
    x = codes[slots, 0].float()
    return x * scale[slots, 0].repeat_interleave(BLOCK, dim=-1)[..., :x.shape[2], None]


def _attend(q, kf, vf, mask):
    """q [n, R, HEADS, HD], kf and vf [n, KVH, T, HD], mask [n, KVH or 1, R, T] -> [n * R, HEADS * HD] BF16."""
    n, R = q.shape[:2]
    qg = q.float().view(n, R, KVH, 2, HD).permute(0, 2, 3, 1, 4)           # [n, KVH, 2, R, HD]
    s = torch.matmul(qg.reshape(n, KVH, 2 * R, HD), kf.transpose(-1, -2)).view(n, KVH, 2, R, -1) * SCALE
    s = torch.where(mask[:, :, None], s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), 0.0, m))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, KVH, 2 * R, -1), vf).view(n, KVH, 2, R, HD) / torch.where(l > 0, l, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(n * R, HEADS * HD).to(torch.bfloat16)


def _plain_attention(st):
    L, n = st["L"], st["pos"].numel()
    slots = st["seq_ids"].long()
    kf, vf = _values(st["k"], st["k_scale"], slots), _values(st["v"], st["v_scale"], slots)
    t = torch.arange(kf.shape[2], device=DEV)
    qpos = st["pos"].long()[:, None] + torch.arange(L, device=DEV)
    mask = t[None, None, None, :] <= qpos[:, None, :, None]
    return _attend(st["q"].view(n, L, HEADS, HD), kf, vf, mask)


def _plain_sparse(st):
    n = st["pos"].numel()
    slots = st["seq_ids"].long()
    blocks = st["blocks"].long()
    t = (blocks[..., None] * BLOCK + torch.arange(BLOCK, device=DEV)).view(n, KVH, -1)
    ok = (blocks >= 0)[..., None].expand(-1, -1, -1, BLOCK).reshape(t.shape) & (t <= st["pos"].long()[:, None, None])
    t = torch.where(ok, t, 0)
    head = torch.arange(KVH, device=DEV)[None, :, None]

    def take(codes, scale):
        x = codes.view(torch.uint8)[slots[:, None, None], 0, head, t].view(E4M3).float()
        return x * scale[slots[:, None, None], 0, head, t // BLOCK][..., None]

    return _attend(st["q"].view(n, 1, HEADS, HD), take(st["k"], st["k_scale"]), take(st["v"], st["v_scale"]),
                   ok[:, :, None])


def _plain_select(st):
    c = st["case"]
    n = st["pos"].numel()
    slots = st["seq_ids"].long()
    bounds = st["k_bounds"][slots, 0].double()                             # [n, KVH, nb, 2, HD]
    q = st["q"].double().view(n, KVH, 2, HD)
    score = torch.matmul(q.clamp(max=0), bounds[..., 0, :].transpose(-1, -2))
    score += torch.matmul(q.clamp(min=0), bounds[..., 1, :].transpose(-1, -2))
    score = score.amax(2) * st["k_scale"][slots, 0].double()
    nb = st["pos"].long() // BLOCK + 1
    idx = torch.arange(score.shape[-1], device=DEV)
    forced = (idx < c["sink"]) | (idx >= nb[:, None, None] - c["recent"])
    return _first_blocks(torch.where(forced, float("inf"), score), nb, c["blocks"])


def _plain_append(st):
    L, p, n = st["L"], st["pos"].long(), st["pos"].numel()
    slots = st["seq_ids"].long()
    max_len = st["k"].shape[3]
    nbt = (L + BLOCK - 2) // BLOCK + 1                                     # blocks that L rows can touch
    b = p[:, None] // BLOCK + torch.arange(nbt, device=DEV)                # [n, nbt]
    t = b[..., None] * BLOCK + torch.arange(BLOCK, device=DEV)             # [n, nbt, BLOCK]
    new = (t >= p[:, None, None]) & (t < p[:, None, None] + L)
    kept = (t < p[:, None, None]) & new.any(-1, keepdim=True)              # what a touched block held
    has_old = (b * BLOCK < p[:, None])[..., None]
    touched = new.any(-1)
    row = (t - p[:, None, None]).clamp(0, L - 1)
    tc, bc = t.clamp(max=max_len - 1), b.clamp(max=st["k_scale"].shape[3] - 1)
    lane = torch.arange(n, device=DEV)[:, None, None]
    head = torch.arange(KVH, device=DEV)
    out = []
    for codes, scale, x, bounds in ((st["k"], st["k_scale"], st["k_new"], st["k_bounds"]),
                                    (st["v"], st["v_scale"], st["v_new"], None)):
        x = x.float().view(n, L, KVH, HD)[lane, row]                       # [n, nbt, BLOCK, KVH, HD]
        use = new[..., None, None]
        fresh = _scale_of(torch.where(use, x.abs(), 0.0).amax((2, 4)))     # [n, nbt, KVH]
        s_old = scale[slots[:, None], 0, :, bc]
        s = torch.where(has_old, torch.maximum(fresh, s_old), fresh)
        shrink = torch.where(has_old, s_old / s, 1.0)
        held = codes.view(torch.uint8)[slots[:, None, None], 0, :, tc].view(E4M3).float()
        held = (held * shrink[:, :, None, :, None]).to(E4M3)
        mixed = torch.where(use, _codes(x, s[:, :, None, :, None]).view(torch.uint8), held.view(torch.uint8))
        put = (new | kept).nonzero(as_tuple=True)
        codes.view(torch.uint8)[slots[put[0]], 0, :, t[put]] = mixed[put]
        at = touched.nonzero(as_tuple=True)
        scale[slots[at[0]], 0, :, b[at]] = s[at]
        if bounds is not None:
            f = mixed.view(E4M3).float()
            lo = torch.where(use, f, float("inf")).amin(2)
            hi = torch.where(use, f, float("-inf")).amax(2)
            was = bounds.view(torch.uint8)[slots[:, None], 0, :, bc].view(E4M3).float()   # [n, nbt, KVH, 2, HD]
            was = (was * shrink[..., None, None]).to(E4M3).float()
            lo = torch.where(has_old[..., None], torch.minimum(lo, was[..., 0, :]), lo)
            hi = torch.where(has_old[..., None], torch.maximum(hi, was[..., 1, :]), hi)
            pair = torch.stack([lo, hi], dim=-2).to(E4M3).view(torch.uint8)
            bounds.view(torch.uint8)[slots[at[0]], 0, :, b[at]] = pair[at]
    return _cache_out(st)


def _cache_out(st):
    return [st["k"], st["v"], st["k_scale"], st["v_scale"], st["k_bounds"]]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op, c = state["case"]["op"], state["case"]
    if not own:
        if op == "append":
            return _plain_append(state)
        if op == "select":
            return _plain_select(state)
        return _plain_sparse(state) if op == "sparse" else _plain_attention(state)
    import n550_qwen3_bringup_handover_b200 as n5
    cache, ids, pos = state["cache"], state["seq_ids"], state["pos"]
    if op == "append":
        n5.kv8_append(cache, state["k_new"], state["v_new"], ids, pos, state["L"], 0)
        return _cache_out(state)
    if op == "select":
        return n5.kv8_select_blocks(state["q"], cache, ids, pos, 0, c["blocks"], c["sink"], c["recent"])
    if op == "sparse":
        return n5.attention_sparse_kv8(state["q"], cache, ids, pos, state["blocks"], 0)
    if op == "decode":
        return n5.attention_decode_kv8(state["q"], cache, ids, pos, 0)
    return n5.attention_prefill_kv8(state["q"], cache, ids, state["L"], c["pos0"], 0)


# ---------------------------------------------------------------------------
# the definitions in 64 bits, a sequence at a time
# ---------------------------------------------------------------------------
def _round_e4m3(y):
    """Nearest e4m3 value to y (ties to even), |y| limited to 448."""
    y = y.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_append(st):
    L = st["L"]
    k, v, ks, vs, kb = (x.double() for x in _cache_out(st))
    for i, (slot, p) in enumerate(zip(st["seq_ids"].tolist(), st["pos"].tolist())):
        for codes, scale, rows, bounds in ((k, ks, st["k_new"], kb), (v, vs, st["v_new"], None)):
            x = rows[i * L:(i + 1) * L].double().view(L, KVH, HD).transpose(0, 1)
            for b in range(p // BLOCK, (p + L - 1) // BLOCK + 1):
                lo, hi = max(p, b * BLOCK), min(p + L, (b + 1) * BLOCK)
                part = x[:, lo - p:hi - p]
                top = part.abs().amax((1, 2)).clamp(min=2.0 ** -130)
                s = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp(min=-126.0))
                s = torch.where(448.0 * s * 0.5 >= top, (s * 0.5).clamp(min=2.0 ** -126), s)
                if p > b * BLOCK:
                    was = scale[slot, 0, :, b].clone()
                    s = torch.maximum(s, was)
                    held = codes[slot, 0, :, b * BLOCK:p]
                    codes[slot, 0, :, b * BLOCK:p] = _round_e4m3(held * (was / s)[:, None, None])
                got = _round_e4m3(part / s[:, None, None])
                codes[slot, 0, :, lo:hi] = got
                scale[slot, 0, :, b] = s
                if bounds is not None:
                    least, most = got.amin(1), got.amax(1)
                    if p > b * BLOCK:
                        old = _round_e4m3(bounds[slot, 0, :, b] * (was / s)[:, None, None])
                        least, most = torch.minimum(least, old[:, 0]), torch.maximum(most, old[:, 1])
                    bounds[slot, 0, :, b] = torch.stack([least, most], dim=1)
    return [k, v, ks, vs, kb]


def _exact_attention(st):
    op, L = st["case"]["op"], st["L"]
    out = torch.zeros((st["pos"].numel() * L, HEADS, HD), dtype=torch.float64, device=DEV)
    for i, (slot, p) in enumerate(zip(st["seq_ids"].tolist(), st["pos"].tolist())):
        for h in range(KVH):
            t = torch.arange(p + L, device=DEV)
            if op == "sparse":
                mine = st["blocks"][i, h].long()
                t = (mine[mine >= 0, None] * BLOCK + torch.arange(BLOCK, device=DEV)).flatten()
                t = t[t <= p]
            kf = st["k"][slot, 0, h].view(torch.uint8)[t].view(E4M3).double() * st["k_scale"][slot, 0, h][t // BLOCK, None].double()
            vf = st["v"][slot, 0, h].view(torch.uint8)[t].view(E4M3).double() * st["v_scale"][slot, 0, h][t // BLOCK, None].double()
            q = st["q"][i * L:(i + 1) * L].double().view(L, HEADS, HD)[:, 2 * h:2 * h + 2]
            s = torch.einsum("lgd,td->glt", q, kf) / math.sqrt(HD)
            s = s.masked_fill(t[None, None, :] > p + torch.arange(L, device=DEV)[None, :, None], float("-inf"))
            out[i * L:(i + 1) * L, 2 * h:2 * h + 2] = torch.einsum("glt,td->lgd", torch.softmax(s, -1), vf)
    return out.view(-1, HEADS * HD)


def _exact_select(st):
    c = st["case"]
    got = torch.full((st["pos"].numel(), KVH, c["blocks"]), -1, dtype=torch.int32)
    for i, (slot, p) in enumerate(zip(st["seq_ids"].tolist(), st["pos"].tolist())):
        nb = p // BLOCK + 1
        for h in range(KVH):
            lo, hi = st["k_bounds"][slot, 0, h, :nb].double().unbind(1)
            q = st["q"][i].double().view(HEADS, HD)[2 * h:2 * h + 2]
            bound = torch.maximum(q[:, None] * lo, q[:, None] * hi).sum(-1).amax(0)
            bound = (bound * st["k_scale"][slot, 0, h, :nb].double()).tolist()
            must = [b for b in range(nb) if b < c["sink"] or b >= nb - c["recent"]]
            rest = sorted((b for b in range(nb) if b not in must), key=lambda b: (-bound[b], b))
            take = sorted((must + rest)[:c["blocks"]])
            got[i, h, :len(take)] = torch.tensor(take, dtype=torch.int32)
    return got


def exact(case, seed):
    if case["op"] == "append" and case["n"] * case["L"] > 40000:
        return None
    st = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(st)
    return _exact_select(st) if case["op"] == "select" else _exact_attention(st)
