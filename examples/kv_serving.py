"""Serving a compressed decoder over an 8-bit paged key/value cache.

A small decoder (12 query heads over one shared key/value head, rotary positions) is compressed by
ElasticBit; ragged prompts are admitted, decoded together one token at a time by replaying a captured
step, one request finishes and its blocks go to a new one.  At the end the logits are compared with
those of the same model over 16-bit keys and values, without a cache.

    python examples/kv_serving.py
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import mlbricks_b200 as mlb  # noqa: E402
from mlbricks_b200.kvcache import KVCache  # noqa: E402

VOCAB, DIM, HEADS, KV_HEADS, LAYERS = 512, 384, 12, 1, 3
HEAD_DIM = DIM // HEADS


def rotate(x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """Rotary positions of x [tokens, heads, HEAD_DIM]."""
    half = HEAD_DIM // 2
    angle = positions[:, None, None] * (10000.0 ** (-torch.arange(half, device=x.device) / half))
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1).to(x.dtype)


class Layer(nn.Module):
    def __init__(self) -> None:
        super().__init__()
        self.q, self.o = nn.Linear(DIM, DIM, bias=False), nn.Linear(DIM, DIM, bias=False)
        self.k, self.v = (nn.Linear(DIM, KV_HEADS * HEAD_DIM, bias=False) for _ in "kv")
        self.up, self.down = nn.Linear(DIM, 4 * DIM), nn.Linear(4 * DIM, DIM)
        self.n1, self.n2 = nn.RMSNorm(DIM), nn.RMSNorm(DIM)

    def forward(self, x, positions, attend):
        h = self.n1(x)
        q = rotate(self.q(h).view(-1, HEADS, HEAD_DIM), positions)
        k = rotate(self.k(h).view(-1, KV_HEADS, HEAD_DIM), positions)
        x = x + self.o(attend(q, k, self.v(h).view(-1, KV_HEADS, HEAD_DIM)).reshape(x.shape))
        return x + self.down(torch.nn.functional.gelu(self.up(self.n2(x))))


class Decoder(nn.Module):
    def __init__(self) -> None:
        super().__init__()
        self.embed = nn.Embedding(VOCAB, DIM)
        self.layers = nn.ModuleList(Layer() for _ in range(LAYERS))
        self.norm, self.head = nn.RMSNorm(DIM), nn.Linear(DIM, VOCAB, bias=False)

    def forward(self, ids, positions=None, cache: KVCache | None = None):
        """Logits of packed tokens [tokens]: over the cache's planned step, or of one whole sequence."""
        if cache is not None:
            positions = cache.step.positions
        elif positions is None:
            ids = ids.reshape(-1)
            positions = torch.arange(ids.numel(), device=ids.device)
        x = self.embed(ids)
        for i, layer in enumerate(self.layers):
            x = layer(x, positions, self.dense if cache is None else lambda q, k, v, i=i: self.cached(cache, i, q, k, v))
        return self.head(self.norm(x))

    @staticmethod
    def cached(cache, layer, q, k, v):
        cache.append(layer, k, v)
        return cache.attention(layer, q)

    @staticmethod
    def dense(q, k, v):
        k, v = (t.repeat_interleave(HEADS // KV_HEADS, 1).float() for t in (k, v))
        score = torch.einsum("ihd,jhd->hij", q.float(), k) / HEAD_DIM**0.5
        score = score.masked_fill(torch.ones_like(score[0], dtype=torch.bool).triu(1), float("-inf"))
        return torch.einsum("hij,jhd->ihd", score.softmax(-1), v).to(q.dtype)


@torch.no_grad()
def serve(steps: int = 24) -> dict:
    torch.manual_seed(0)
    model = Decoder().half().cuda().eval()
    calibration = torch.randint(VOCAB, (64,), device="cuda")
    mlb.ElasticBit.compress(model, calibrationData=calibration, threshold=0.01, backend="native")

    prompts = [5, 130, 64, 333]
    rows = len(prompts)
    cache = KVCache(LAYERS, blocks=40, kv_heads=KV_HEADS, head_dim=HEAD_DIM, requests=rows, max_length=640, block_size=32)
    texts = [torch.randint(VOCAB, (n,), device="cuda") for n in prompts]

    def admit(new):
        """Prompts of the rows whose new tokens are more than 0; their first answers."""
        step = cache.plan(new)
        logits = model(torch.cat([texts[i][-n:] for i, n in enumerate(new) if n > 0]), cache=cache)
        last = step.starts[1:].long() - 1
        for i, n in enumerate(new):
            if n > 0:
                texts[i] = torch.cat([texts[i], logits[last[i]].argmax().view(1)])

    admit(prompts)

    # one decode step of every row, captured once
    ids = torch.stack([t[-1] for t in texts])
    ones = torch.ones(rows, dtype=torch.int32, device="cuda")

    def decode():
        cache.plan(ones, tokens=rows, max_new=1)
        missing.add_(cache.ring[2])
        logits.copy_(model(ids, cache=cache))
        ids.copy_(logits.argmax(-1))

    logits = torch.empty(rows, VOCAB, dtype=torch.float16, device="cuda")
    missing = torch.zeros((), dtype=torch.int64, device="cuda")  # blocks that were not there, over all steps
    state = [t.clone() for t in (cache.lengths, cache.ring, cache.tables, cache.free, ids, missing)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode()  # warms up; its tokens are planned again below
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decode()
    for now, then in zip((cache.lengths, cache.ring, cache.tables, cache.free, ids, missing), state):
        now.copy_(then)

    def run(n):
        for _ in range(n):
            graph.replay()
            for i in range(rows):
                texts[i] = torch.cat([texts[i], ids[i].view(1)])

    run(steps // 2)
    # request 1 is done; its blocks serve a new prompt in the same row
    cache.plan([-1 if i == 1 else 0 for i in range(rows)])
    texts[1] = torch.randint(VOCAB, (200,), device="cuda")
    admit([200 if i == 1 else 0 for i in range(rows)])
    ids.copy_(torch.stack([t[-1] for t in texts]))
    run(steps - steps // 2)

    errors = []
    for i in range(rows):
        want = model(texts[i][:-1])[-1].float()
        errors.append(float((logits[i].float() - want).norm() / want.norm()))
    return {"lengths": cache.lengths.tolist(), "texts": [t.numel() for t in texts], "errors": errors, "missing": int(missing),
            "free": int(cache.ring[1] - cache.ring[0])}


if __name__ == "__main__":
    if not torch.cuda.is_available():
        sys.exit("needs a CUDA device")
    result = serve()
    print("tokens held:", result["lengths"], " free blocks:", result["free"])
    print("logits against 16-bit keys and values, relative:", ["%.4f" % e for e in result["errors"]])
