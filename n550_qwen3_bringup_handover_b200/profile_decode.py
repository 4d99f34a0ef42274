"""Run greedy decode steps of the random-init model on a bounded case (for
profilers): n_seqs sequences with a ctx-token prefilled context, then `steps`
eager decode steps (one kernel sequence per step, no CUDA graph). With --kv8, over
the 8-bit KV cache. With --time, report the device time per step instead (CUDA
events over `steps` replays of the captured step, median of 5 such runs after one).

    python -m n550_qwen3_bringup_handover_b200.profile_decode --seqs 64 --ctx 1024 --steps 2
    python -m n550_qwen3_bringup_handover_b200.profile_decode --seqs 64 --ctx 1024 --steps 24 --kv8 --time
"""
from __future__ import annotations

import argparse

import torch

import n550_qwen3_bringup_handover_b200 as n5


def timed(m, cur, seq, ctx, steps):
    """Median us per step of `steps` greedy steps from position ctx."""
    out = torch.empty((steps, len(seq)), dtype=torch.int32, device="cuda")
    tok, pos = cur.clone(), torch.empty_like(seq)
    us = []
    for run in range(6):
        tok.copy_(cur)
        pos.fill_(ctx)
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        m.decode_steps(tok, seq, pos, steps, out)
        e1.record()
        e1.synchronize()
        if run:                               # the first one captures the step
            us.append(e0.elapsed_time(e1) / steps * 1e3)
    return sorted(us)[len(us) // 2]


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--seqs", type=int, default=64)
    ap.add_argument("--ctx", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=2)
    ap.add_argument("--kv8", action="store_true")
    ap.add_argument("--time", action="store_true")
    a = ap.parse_args()
    m = n5.Model(seed=0, max_seqs=a.seqs, max_len=a.ctx + a.steps + 1, max_tokens=a.seqs * a.ctx, kv8=a.kv8)
    tok = torch.from_numpy(n5.synth_tokens(a.seqs * a.ctx, 0, 0x544F4B).reshape(a.seqs, a.ctx)).cuda()
    seq = torch.arange(a.seqs, dtype=torch.int32, device="cuda")
    nxt = torch.empty(a.seqs, dtype=torch.int32, device="cuda")
    m.prefill(tok, seq, 0, None, nxt)
    if a.time:
        us = timed(m, nxt, seq, a.ctx, a.steps)
        print(f"seqs={a.seqs} ctx={a.ctx} {'8-bit' if a.kv8 else 'BF16'} KV cache: {us:.1f} us per step")
    pos = torch.full((a.seqs,), a.ctx, dtype=torch.int32, device="cuda")
    for _ in range(0 if a.time else a.steps):
        cur = nxt.clone()
        m.decode(cur, seq, pos, None, nxt)
        pos += 1
    torch.cuda.synchronize()
    n5.check(n5.device_status(), "device status")
    print("ok", nxt[:4].tolist())
    m.close()


if __name__ == "__main__":
    main()
