"""The 8-bit KV cache's definitions in binary64 on the CPU, one sequence at a
time: what tests/test_kv8*.py compare the kernels with."""
import torch

BLOCK, KVH, HEADS, HD = 64, 8, 16, 128
E4 = torch.float8_e4m3fn
# (index of) the finite non-negative e4m3 values, ascending: codes 0x00 .. 0x7E
POS = torch.tensor([(m / 8 if e == 0 else 1 + m / 8) * 2.0 ** ((e or 1) - 7)
                    for e in range(16) for m in range(8) if (e, m) != (15, 7)], dtype=torch.float64)


def values(codes):
    """e4m3 codes (uint8) -> binary64, from the format's definition."""
    c = codes.to(torch.int64)
    mag = torch.cat([POS, torch.tensor([float("nan")], dtype=torch.float64)])[c & 127]
    return torch.where((c & 128) != 0, -mag, mag)


def round_codes(y):
    """Nearest e4m3 code (uint8) to binary64 y: ties to the even code, beyond 448
    the largest, NaN the NaN code."""
    a = y.abs().nan_to_num(nan=0.0, posinf=1e300).clamp(max=448.0)
    hi = torch.searchsorted(POS, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    below, above = a - POS[lo], POS[hi] - a
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    code = torch.where(up, hi, lo) | torch.where(torch.signbit(y), 128, 0)
    return torch.where(y.isnan(), torch.tensor(127), code).to(torch.uint8)


def scale_for(x):
    """Smallest power of two s >= 2^-126 with |x| <= 448 s over the finite values."""
    a = x[torch.isfinite(x)].abs()
    top = float(a.max()) if a.numel() else 0.0
    e = -126
    while 448.0 * 2.0 ** e < top:
        e += 1
    return 2.0 ** e


class Cache:
    """codes uint8, scales float64; mirrors n550_kv8_cache for one layer."""

    def __init__(self, n_slots, max_len):
        nb = -(-max_len // BLOCK)
        self.n_slots, self.max_len = n_slots, max_len
        self.code = {w: torch.zeros((n_slots, KVH, max_len, HD), dtype=torch.uint8) for w in "kv"}
        self.scale = {w: torch.zeros((n_slots, KVH, nb), dtype=torch.float64) for w in "kv"}
        self.bounds = torch.zeros((n_slots, KVH, nb, 2, HD), dtype=torch.uint8)

    @classmethod
    def of(cls, cache, layer):
        """A copy of a device KV8Cache's layer."""
        c = cls(cache.n_slots, cache.max_len)
        c.code = {"k": cache.k[:, layer].view(torch.uint8).cpu(), "v": cache.v[:, layer].view(torch.uint8).cpu()}
        c.scale = {"k": cache.k_scale[:, layer].double().cpu(), "v": cache.v_scale[:, layer].double().cpu()}
        if cache.k_bounds is not None:
            c.bounds = cache.k_bounds[:, layer].view(torch.uint8).cpu()
        return c

    def append(self, k, v, seq_ids, pos, L):
        for i, (slot, p) in enumerate(zip(seq_ids, pos)):
            if not 0 <= slot < self.n_slots or p < 0 or p + L > self.max_len:
                continue
            for w, rows in (("k", k), ("v", v)):
                x = rows[i * L:(i + 1) * L, :KVH * HD].double().view(L, KVH, HD)
                for h in range(KVH):
                    for b in range(p // BLOCK, (p + L - 1) // BLOCK + 1):
                        self._block(w, slot, h, b, p, L, x[:, h])

    def _block(self, w, slot, h, b, p, L, x):
        lo, hi = max(p, b * BLOCK), min(p + L, (b + 1) * BLOCK)
        part = x[lo - p:hi - p]
        s, code = scale_for(part), self.code[w][slot, h]
        if p > b * BLOCK:
            old = float(self.scale[w][slot, h, b])
            s = max(s, old)
            if s > old:
                code[b * BLOCK:p] = round_codes(values(code[b * BLOCK:p]) * (old / s))
        code[lo:hi] = round_codes(part / s)
        self.scale[w][slot, h, b] = s
        if w == "k":
            got = values(code[lo:hi]).nan_to_num(nan=0.0)
            least, most = got.amin(0), got.amax(0)
            if p > b * BLOCK:
                was = values(round_codes(values(self.bounds[slot, h, b]) * (old / s)))
                least, most = torch.minimum(least, was[0]), torch.maximum(most, was[1])
            self.bounds[slot, h, b] = round_codes(torch.stack([least, most]))

    def dequant(self, w, slot, h, t):
        return values(self.code[w][slot, h, t]) * self.scale[w][slot, h, t // BLOCK, None]

    def context(self, slot, pos):
        return 0 if not 0 <= slot < self.n_slots or pos < 0 else min(pos, self.max_len - 1) + 1

    def attend(self, q, seq_ids, pos, L=1, blocks=None, floor=2.0 ** -15):
        """(out, mass) [n * L, 2048] binary64: mass_d = sum_t (softmax_t + floor) |v_td|,
        the scale that a rounding of the weights acts on: a weight rounded
        relative to itself moves out by that part of the first term, and one
        rounded to a multiple of 2^-25 of the largest weight (small ones are; half
        a step is 2^-26, and the weights' sum is at least the largest) by at most
        2^-26 |v_td|, which 2^-11 of the second term covers. (Where V's block scales
        differ the multiple is up to 2^-22, and floor has to be 2^-12.)"""
        n = len(seq_ids)
        q = q[:, :HEADS * HD].double().cpu().view(n, L, HEADS, HD)
        out = torch.zeros((n, L, HEADS, HD), dtype=torch.float64)
        mass = torch.zeros_like(out)
        for i, (slot, p) in enumerate(zip(seq_ids, pos)):
            for h in range(KVH):
                for j in range(L):
                    length = self.context(slot, p + j if p >= 0 else p)
                    t = torch.arange(length)
                    if blocks is not None:
                        mine = [b for b in blocks[i][h] if b >= 0]
                        t = torch.cat([torch.arange(b * BLOCK, (b + 1) * BLOCK) for b in mine] or [t[:0]])
                        t = t[t < length]
                    if not t.numel():
                        continue
                    k, v = self.dequant("k", slot, h, t), self.dequant("v", slot, h, t)
                    w = torch.softmax(q[i, j, 2 * h:2 * h + 2] @ k.T * 0.08838834764831845, -1)
                    out[i, j, 2 * h:2 * h + 2] = w @ v
                    mass[i, j, 2 * h:2 * h + 2] = (w + floor) @ v.abs()
        return out.view(n * L, -1), mass.view(n * L, -1)

    def select(self, q, seq_ids, pos, n_select, n_sink, n_recent):
        n = len(seq_ids)
        q = q[:, :HEADS * HD].double().cpu().view(n, HEADS, HD)
        got = torch.full((n, KVH, n_select), -1, dtype=torch.int32)
        for i, (slot, p) in enumerate(zip(seq_ids, pos)):
            nb = -(-self.context(slot, p) // BLOCK)
            for h in range(KVH):
                score = []
                for b in range(nb):
                    lo, hi = values(self.bounds[slot, h, b])
                    g = q[i, 2 * h:2 * h + 2]
                    top = torch.maximum(g * lo, g * hi).sum(-1)
                    top = float("-inf") if top.isnan().all() else float(top[~top.isnan()].max())
                    score.append(top * float(self.scale["k"][slot, h, b]))
                must = [b for b in range(nb) if b < n_sink or b >= nb - n_recent]
                rest = sorted(set(range(nb)) - set(must), key=lambda b: (-score[b], b))
                take = sorted((must + rest)[:n_select])
                got[i, h, :len(take)] = torch.tensor(take, dtype=torch.int32)
        return got
