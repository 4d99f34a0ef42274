"""What the 8-bit KV cache costs the model: its logits against a plain FP32 forward whose K
and V are rounded to the cache's codes, and against one whose are not; and the
generation loops over it.

How near. e: the error in the mean square that the codes make in the plain forward's
logits (measured here, with and without them). Per element it is 2.5 % of K and V: half
a step is 2^-4 of a binade, so (2^-3)^2 / 12 in the mean square, over 2.16 for values
uniform in the logarithm. The library's rows differ from the plain ones by at most the
1e-2 that its fast mode is held to, and where an element then falls on the other side of
a border between codes, it moves by a step: a difference d does that to 0.8 * 1.44 d / 2^-3
= 9.2 d of them, and (2^-3)^2 * 9.2 d / 2.16 is (2.6 %)^2 for d = 1e-2. These errors enter
where e's do and grow as they do, so they are at most 2.6 / 2.45 = 1.06 e in the logits:
1.15 e + 1e-2 allows for 2 % of fluctuation in either (1024 dimensions of a row), and for
the library's own difference without codes. To the forward without codes it is e more."""
import numpy as np
import pytest
import torch

import n550_qwen3_bringup_handover_b200 as n5
import oracle
from kv8_oracle import BLOCK
from tests.conftest import GOLDEN

pytestmark = pytest.mark.gpu
ROUTES = 2.5e-2        # largest logit error between two routes over the 8-bit cache (tests/test_kv8_model_gpu.py)


def toks(n, seed):
    return torch.from_numpy(oracle.synth_tokens(n, seed, 0x544F4B)).cuda()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rms(x):
    return float(x.double().square().mean().sqrt())


@pytest.fixture(scope="module")
def weights(cuda):
    m = n5.Model(seed=0, max_seqs=1, max_len=8, max_tokens=8)
    shapes = [(2048, 1024), (1024, 1024), (1024, 1024), (128,), (128,), (1024, 2048), (1024,), (-1, 1024),
              (-1, 1024), (1024, -1)]
    layer = [(1024,)] + shapes

    def get(i, shape):
        return torch.from_numpy(m.weight_bits(i).view(np.int16)).view(torch.bfloat16).cuda().float().view(shape)

    w = dict(embed=get(0, (151936, 1024)), final=get(1 + 28 * 11, (1024,)),
             layers=[[get(1 + 11 * l + k, layer[k]) for k in range(11)] for l in range(28)])
    m.close()
    yield w


def norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w


def coded(x):
    """[n, heads, T, 128] as the cache holds them: BF16, then e4m3 with a power of two for 64 positions."""
    n, h, T, d = x.shape
    x = torch.nn.functional.pad(x.bfloat16().float(), (0, 0, 0, -T % BLOCK)).view(n, h, -1, BLOCK, d)
    top = x.abs().amax((-1, -2), keepdim=True)
    s = torch.exp2(torch.ceil(torch.log2(top.double() / 448)).clamp(min=-126)).float()
    return ((x / s).clamp(-448, 448).to(torch.float8_e4m3fn).float() * s).view(n, h, -1, d)[:, :, :T]


def plain(w, t, first, codes):
    """FP32 logits [n, T - first, 151936] of token rows t [n, T] at positions first .."""
    n, T = t.shape
    x = w["embed"][t.long()]
    f = 1e6 ** (-torch.arange(64, device="cuda", dtype=torch.float64) / 64)
    ang = torch.arange(T, device="cuda", dtype=torch.float64)[:, None] * f
    cos, sin = ang.cos().float(), ang.sin().float()

    def heads(y, k):
        return y.view(n, T, k, 128).transpose(1, 2)

    def rope(y):
        a, b = y[..., :64], y[..., 64:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    later = torch.ones((T, T), dtype=torch.bool, device="cuda").triu(1)
    for n0, wq, wk, wv, qn, kn, wo, n1, wg, wu, wd in w["layers"]:
        y = norm(x, n0)
        q, k, v = rope(norm(heads(y @ wq.T, 16), qn)), rope(norm(heads(y @ wk.T, 8), kn)), heads(y @ wv.T, 8)
        if codes:
            k, v = coded(k), coded(v)
        k, v = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
        s = (q @ k.transpose(-1, -2) * 128 ** -0.5).masked_fill(later, float("-inf"))
        x = x + (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(n, T, -1) @ wo.T
        y = norm(x, n1)
        x = x + (torch.nn.functional.silu(y @ wg.T) * (y @ wu.T)) @ wd.T
    return norm(x[:, first:], w["final"]) @ w["embed"].T


@pytest.mark.parametrize("n_seqs,L", [(1, 1), (1, 5), (1, 200), (6, 100), (20, 30), (70, 16), (5, 259)])
def test_logits_are_those_of_rounded_keys_and_values(weights, n_seqs, L):
    """A prefill and six decode steps of the same tokens (every q/k/v route and both
    prefill attentions)."""
    steps = 6
    t = toks(n_seqs * (L + steps), 91).view(n_seqs, L + steps)
    ids = torch.randperm(n_seqs, generator=torch.Generator().manual_seed(L)).to(torch.int32).cuda()

    def library(kv8):
        m = n5.Model(seed=0, max_seqs=n_seqs, max_len=L + steps + 3, max_tokens=n_seqs * L + 8, kv8=kv8)
        try:
            out = [torch.empty((n_seqs, 151936), dtype=torch.float32, device="cuda") for _ in range(steps + 1)]
            m.prefill(t[:, :L].contiguous(), ids, 0, out[0])
            for j in range(steps):
                m.decode(t[:, L + j].contiguous(), ids, i32([L + j] * n_seqs), out[1 + j])
            torch.cuda.synchronize()
            return torch.stack(out, 1)
        finally:
            m.close()

    got, bf16 = library(True), library(False)
    assert n5.device_status() == n5.OK
    exact, rounded = plain(weights, t, L - 1, False), plain(weights, t, L - 1, True)
    size = rms(exact)
    e = rms(rounded - exact) / size
    near, far, cost = rms(got - rounded) / size, rms(got - exact) / size, rms(got - bf16) / size
    worst = float(((got - bf16).abs().amax(-1) / bf16.abs().amax(-1)).max())
    print(f"{n_seqs} x {L}: codes {e:.4f} in the plain forward; library to it {near:.4f}, to the one without codes {far:.4f}, "
          f"to its BF16 cache {cost:.4f} (largest logit error {worst:.4f} of the largest logit; "
          f"BF16 cache to plain {rms(bf16 - exact) / size:.4f}; same choice {float((got.argmax(-1) == bf16.argmax(-1)).float().mean()):.3f})")
    assert near <= 1.15 * e + 1e-2
    assert far <= 2.15 * e + 1e-2


def greedy_by(m, prompt, ids):
    """Every id is the largest logit after those before it, or within two routes' difference
    of it: all rows' logits of the whole sequence on the same model."""
    seq = np.concatenate([np.asarray(prompt, np.int32), np.asarray(ids, np.int32)])[:-1]
    rows = np.concatenate([m.forward_rows(seq[at:at + 100], at, want_logits=True)[1] for at in range(0, len(seq), 100)])
    rows = rows[len(prompt) - 1:]
    assert len(rows) == len(ids)
    for i, (row, t) in enumerate(zip(rows, ids)):
        assert row.max() - row[t] <= 2 * ROUTES * np.abs(row).max(), (i, int(t), int(row.argmax()))


def test_generate_lookup(cuda):
    """Plain and with drafts. Rejected drafts may raise the scale of the block that they
    were appended to, which rounds its held codes anew, and rows verified together are
    appended together: the drafted ids are greedy ids within the routes' difference, not
    the plain ones bit for bit."""
    prompt = np.load(GOLDEN / "greedy_ref.npz")["prompt"]
    m = n5.Model(seed=0, max_seqs=1, max_len=256, max_tokens=128, kv8=True)
    try:
        plain, st0 = m.generate_lookup(prompt, 64, max_draft=0, eos=())
        again, _ = m.generate_lookup(prompt, 64, max_draft=0, eos=())
        spec, st = m.generate_lookup(prompt, 64, max_draft=127, eos=())
        rejected = st["drafted"] - st["accepted"]
        assert len(plain) == len(spec) == 64 and np.array_equal(plain, again)
        assert st0 == {"rounds": 64, "drafted": 0, "accepted": 0}
        assert st["rounds"] + st["accepted"] == 64 and st["accepted"] > 0 and rejected > 0
        greedy_by(m, prompt, plain)
        greedy_by(m, prompt, spec)
        stop = int(plain[5])
        if stop not in plain[:5].tolist():
            short, _ = m.generate_lookup(prompt, 64, max_draft=0, eos=(stop,))
            assert np.array_equal(short, plain[:5])
    finally:
        m.close()
    assert n5.device_status() == n5.OK


@pytest.mark.skipif(not oracle.tokenizer_available(), reason="oracle/_ref not built")
def test_chat(cuda):
    prompt = "你好，请介绍一下你自己"
    tok = n5.Tokenizer(oracle.TOK_PATH)
    m = n5.Model(seed=0, max_seqs=1, max_len=256, max_tokens=128, kv8=True)
    try:
        for draft in (0, 127):
            text, ids = m.chat(tok, prompt, max_new=16, max_draft=draft)
            assert text == tok.decode(ids)
            if len(ids):
                greedy_by(m, tok.chat(prompt), ids)
    finally:
        m.close()
    assert n5.device_status() == n5.OK
