"""Samples of one prompt over cache blocks that they share.

The decoder of kv_serving.py reads a prompt once; five more rows fork it, so that its full blocks are held once,
and all six are sampled together, one token at a time.  (Attention would read the shared blocks once for all rows if they were
many or long; for so few tokens ``takes_prefixes`` says that each row by itself is faster.)
At the end the cache is compacted, and the logits are compared with those of the same model over 16-bit keys and values, without
a cache.

    python examples/kv_samples.py
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))

from kv_serving import HEAD_DIM, KV_HEADS, LAYERS, VOCAB, Decoder, mlb  # noqa: E402

from mlbricks_b200.kvshare import SharedKVCache  # noqa: E402


@torch.no_grad()
def serve(steps: int = 20, samples: int = 6) -> dict:
    torch.manual_seed(0)
    model = Decoder().half().cuda().eval()
    mlb.ElasticBit.compress(model, calibrationData=torch.randint(VOCAB, (64,), device="cuda"), threshold=0.01, backend="native")
    cache = SharedKVCache(LAYERS, blocks=60, kv_heads=KV_HEADS, head_dim=HEAD_DIM, requests=samples, max_length=640, block_size=32)

    prompt = torch.randint(VOCAB, (333,), device="cuda")
    cache.plan([prompt.numel()] + [0] * (samples - 1))
    logits = model(prompt, cache=cache)[-1:].expand(samples, VOCAB)
    cache.fork([0] * samples)
    texts = prompt.expand(samples, -1)
    for _ in range(steps):
        ids = torch.multinomial(logits.float().softmax(-1), 1)
        texts = torch.cat([texts, ids], 1)
        cache.plan([1] * samples)
        logits = model(ids[:, 0], cache=cache)

    done = cache.compact()
    held = cache.pools[0].blocks - int(done.ring[1])
    errors = []
    for i in range(samples):
        want = model(texts[i])[-1].float()
        errors.append(float((logits[i].float() - want).norm() / want.norm()))
    return {"lengths": cache.lengths.tolist(), "held": held, "errors": errors,
            "compacted": sorted({x for x in cache.tables.flatten().tolist() if x >= 0})}


if __name__ == "__main__":
    if not torch.cuda.is_available():
        sys.exit("needs a CUDA device")
    result = serve()
    print("tokens held:", result["lengths"], " blocks:", result["held"])
    print("logits against 16-bit keys and values, relative:", ["%.4f" % e for e in result["errors"]])
