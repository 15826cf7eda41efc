"""A small decoder with a sliding attention window, trained and then sampled from.

Each block is: layer norm, one packed q / k / v projection, sliding-window attention with sinks,
output projection, then residual + dropout(projection + bias) in one call; and the same around a
gelu MLP. Training runs the package's mixed-precision tail (GradScaler, clip_grad_norm_, AdamW with a
bf16 model copy) and its cross-entropy; dropout masks come from (seed, offset), one offset per
call, so nothing of them is stored and a step can be repeated. Generation keeps a key / value
cache and takes one token at a time through ``sliding_window_attention_step``.

    python examples/windowed_decoder.py [steps]
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import namitorch_b200 as nt  # noqa: E402
from namitorch_b200.backends import get_backend  # noqa: E402
from namitorch_b200.nn import functional as F  # noqa: E402
from namitorch_b200.optim import AdamW, clip_grad_norm_  # noqa: E402

VOCAB, WIDTH, HEADS, KV_HEADS, LAYERS = 64, 256, 4, 2, 2
DIM = WIDTH // HEADS
WINDOW, SINKS, DROPOUT, SEED = 24, 2, 0.1, 1234
QKV = (HEADS + 2 * KV_HEADS) * DIM


class LayerNorm(torch.autograd.Function):
    """The package's layer norm with its input and affine gradients."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        x = x.contiguous()
        y, statistics = get_backend(x).normalization.run("layer_norm", (x, weight, bias), eps=1e-5)
        ctx.save_for_backward(x, weight, statistics)
        return y

    @staticmethod
    def backward(ctx, grad):
        x, weight, statistics = ctx.saved_tensors
        return get_backend(x).normalization.run("layer_norm_backward", (x, weight, grad.contiguous(), statistics))


class BiasGelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias):
        ctx.save_for_backward(x, bias)
        return get_backend(x).fused.run("bias_gelu_tanh", (x, bias))

    @staticmethod
    def backward(ctx, grad):
        x, bias = ctx.saved_tensors
        dx = get_backend(x).fused.run("bias_gelu_tanh_backward", (x, bias, grad.contiguous()))
        return dx, dx.flatten(0, -2).float().sum(0).to(bias.dtype)


def init_parameters(device, tokens: int, seed: int = 0) -> dict[str, torch.nn.Parameter]:
    g = torch.Generator().manual_seed(seed)
    p = {"tok_emb": (VOCAB, WIDTH), "pos_emb": (tokens, WIDTH), "ln_f.w": (WIDTH,), "ln_f.b": (WIDTH,)}
    for i in range(LAYERS):
        p |= {f"h{i}.ln1.w": (WIDTH,), f"h{i}.ln1.b": (WIDTH,), f"h{i}.qkv.W": (QKV, WIDTH), f"h{i}.qkv.b": (QKV,),
              f"h{i}.proj.W": (WIDTH, WIDTH), f"h{i}.proj.b": (WIDTH,), f"h{i}.ln2.w": (WIDTH,), f"h{i}.ln2.b": (WIDTH,),
              f"h{i}.fc.W": (4 * WIDTH, WIDTH), f"h{i}.fc.b": (4 * WIDTH,), f"h{i}.fc2.W": (WIDTH, 4 * WIDTH),
              f"h{i}.fc2.b": (WIDTH,)}
    out = {}
    for name, shape in p.items():
        norm_weight = name.split(".")[-2:][0].startswith("ln") and name.endswith(".w")
        value = torch.ones(shape) if norm_weight else torch.zeros(shape) if len(shape) == 1 else torch.randn(
            shape, generator=g) * 0.05
        out[name] = torch.nn.Parameter(value.to(device))
    return out


def split_heads(packed):
    """[batch, tokens, QKV] -> query, key, value as views [batch, heads, tokens, DIM]."""
    return (t.transpose(1, 2) for t in packed.unflatten(-1, (HEADS + 2 * KV_HEADS, DIM)).split((HEADS, KV_HEADS, KV_HEADS), 2))


def block(p, i, x, attend, offset, training):
    """One decoder block on [batch, tokens, WIDTH]; ``offset`` numbers its two dropout calls."""
    h = f"h{i}."
    drop = dict(p=DROPOUT, seed=SEED, training=training)
    packed = F.linear(LayerNorm.apply(x, p[h + "ln1.w"], p[h + "ln1.b"]), p[h + "qkv.W"], p[h + "qkv.b"])
    heads = attend(i, packed).transpose(1, 2).flatten(2)
    x = F.dropout(F.linear(heads, p[h + "proj.W"]), bias=p[h + "proj.b"], residual=x, offset=offset, **drop)
    y = F.linear(LayerNorm.apply(x, p[h + "ln2.w"], p[h + "ln2.b"]), p[h + "fc.W"])
    y = F.linear(BiasGelu.apply(y, p[h + "fc.b"]), p[h + "fc2.W"])
    return F.dropout(y, bias=p[h + "fc2.b"], residual=x, offset=offset + 1, **drop)


def logits(p, tokens, attend, first=0, step=0, training=False):
    x = p["tok_emb"][tokens] + p["pos_emb"][first:first + tokens.shape[1]]
    for i in range(LAYERS):
        x = block(p, i, x, attend, 2 * (step * LAYERS + i), training)
    return F.linear(LayerNorm.apply(x, p["ln_f.w"], p["ln_f.b"]), p["tok_emb"])


def full_attention(_, packed):
    q, k, v = split_heads(packed)
    return F.sliding_window_attention(q, k, v, window=WINDOW, sinks=SINKS)


class Cache:
    """Keys and values of every layer, and how many of each sequence are there."""

    def __init__(self, batch, capacity, dtype, device):
        self.k = torch.zeros(LAYERS, batch, KV_HEADS, capacity, DIM, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)

    def prompt(self, i, packed):
        """Attention over the prompt, which fills the cache."""
        q, k, v = split_heads(packed)
        n = k.shape[2]
        self.k[i, :, :, :n], self.v[i, :, :, :n] = k, v
        return F.sliding_window_attention(q, self.k[i, :, :, :n], self.v[i, :, :, :n], window=WINDOW, sinks=SINKS)

    def step(self, i, packed):
        """Attention of one new token, whose place the caller has counted in ``lengths``."""
        q, k, v = split_heads(packed)
        rows = torch.arange(k.shape[0], device=k.device)
        self.k[i][rows, :, (self.lengths - 1).long()], self.v[i][rows, :, (self.lengths - 1).long()] = k[:, :, 0], v[:, :, 0]
        out = F.sliding_window_attention_step(q[:, :, 0], self.k[i], self.v[i], self.lengths, window=WINDOW, sinks=SINKS)
        return out.unsqueeze(2)


def batch_of(step, batch, tokens, device):
    """Sequences that repeat a random pattern of 8 tokens: the window is enough to predict them."""
    g = torch.Generator().manual_seed(step)
    return torch.randint(0, VOCAB, (batch, 8), generator=g).repeat(1, tokens // 8 + 1)[:, :tokens + 1].to(device)


def train(steps=60, batch=16, tokens=64, device="cuda"):
    p = init_parameters(device, tokens + 64)
    optimizer = AdamW([{"params": [t for t in p.values() if t.dim() > 1], "weight_decay": 0.1},
                       {"params": [t for t in p.values() if t.dim() == 1], "weight_decay": 0.0}],
                      lr=2e-3, model_dtype=torch.bfloat16)
    scaler = nt.GradScaler(init_scale=1024.0)
    losses = []
    for step in range(steps):
        data = batch_of(step, batch, tokens, device)
        optimizer.zero_grad()
        loss = F.cross_entropy(logits(p, data[:, :-1], full_attention, step=step, training=True), data[:, 1:])
        scaler.scale(loss).backward()
        scaler.unscale_(optimizer)
        clip_grad_norm_(list(p.values()), 1.0)
        scaler.step(optimizer)
        scaler.update()
        losses.append(loss.item())
        F.check_attention(device)
    return p, losses


@torch.no_grad()
def generate(p, prompt, count):
    """(tokens, the logits of every new position), greedily."""
    cache = Cache(prompt.shape[0], prompt.shape[1] + count, p["tok_emb"].dtype, prompt.device)
    out = logits(p, prompt, cache.prompt)[:, -1]
    cache.lengths.fill_(prompt.shape[1])
    tokens, scores = prompt, []
    for n in range(count):
        scores.append(out)
        tokens = torch.cat([tokens, out.argmax(-1, keepdim=True)], 1)
        cache.lengths += 1
        out = logits(p, tokens[:, -1:], cache.step, first=prompt.shape[1] + n)[:, -1]
    return tokens, torch.stack(scores, 1)


def main(steps=60):
    p, losses = train(steps)
    prompt = batch_of(10_000, 4, 40, "cuda")[:, :-1]
    tokens, _ = generate(p, prompt, 24)
    F.check_attention(tokens.device)
    right = float((tokens[:, 40:] == batch_of(10_000, 4, 64, "cuda")[:, 40:64]).float().mean())
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {len(losses)} steps; {100 * right:.0f}% of 96 generated tokens "
          "continue the pattern")
    return losses, right


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 60)
