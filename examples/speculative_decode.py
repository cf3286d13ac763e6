"""Speculative decoding: the segment-tree engine drafts, the dense model verifies over the 8-bit paged cache.

    python examples/speculative_decode.py [--batch 8] [--prompt 1000] [--tokens 64] [--draft 4] [--temperature 1.0]

Random-init weights of a small GPT (the drafts stand about as often as the sparse attention's distribution agrees with the
dense one's); with a checkpoint, use Decoder.from_checkpoint and weights_from_ours of its state dict for the two."""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from treeattn_b200.config import Config  # noqa: E402
from treeattn_b200.engine import Decoder, weights_from_ours  # noqa: E402
from treeattn_b200.model import GPT  # noqa: E402
from treeattn_b200.speculative import PagedDecoder, SpeculativeDecoder  # noqa: E402


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument('--batch', type=int, default=8)
    ap.add_argument('--prompt', type=int, default=1000)
    ap.add_argument('--tokens', type=int, default=64)
    ap.add_argument('--draft', type=int, default=4)
    ap.add_argument('--temperature', type=float, default=1.0)
    a = ap.parse_args()
    torch.manual_seed(0)
    cfg = Config(attn='seg', vocab_size=8192, seq_len=4096, n_layer=6, n_head=6, n_embd=384, wmax=8, beam=8, local=128,
                 neighbors=False, leaf=64)
    W = weights_from_ours(GPT(cfg).state_dict(), cfg)
    args = (W, cfg.n_layer, cfg.n_head, cfg.n_embd)
    draft = Decoder(*args, cfg.seq_len, 'seg', cfg, 'cuda', batch=a.batch, dtype=torch.bfloat16)
    target = PagedDecoder(*args, batch=a.batch, max_len=cfg.seq_len)
    dec = SpeculativeDecoder(draft, target, a.draft, a.temperature)
    prompts = torch.randint(cfg.vocab_size, (a.batch, a.prompt))
    out = [[int(t)] for t in dec.prefill(prompts)]
    dec.step()  # (captures the drafting graph)
    torch.cuda.synchronize()
    t, steps = time.perf_counter(), 0
    while min(map(len, out)) < a.tokens:
        for o, new in zip(out, dec.step()):
            o.extend(new)
        steps += 1
    torch.cuda.synchronize()
    s = time.perf_counter() - t
    print('%d sequences, %d rounds: %.2f tokens a round and sequence, %.0f tokens/s, %.0f %% of the drafts stood' % (
        a.batch, steps, sum(map(len, out)) / a.batch / steps, sum(map(len, out)) / s, 100 * dec.accepted / dec.drafted))


if __name__ == '__main__':
    main()
