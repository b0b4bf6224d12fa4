"""A text encoder whose attention blocks' projections speak in many voices.

Packed phoneme sequences, each in a voice of its own, go through one block:

    qkv = x Wqkv^T  + the row's voice's low-rank adapters (three units)
    o   = attention inside each utterance
    y   = x + dropout(o Wo^T + the voice's adapters + bias)

``TextBlock.forward`` and ``backward`` train the voices' adapters (the shared
projections stay as they are); ``TextBlock.step`` takes one new token for each
utterance over a key and value cache.

``TextModel`` stacks such blocks from token ids on, each between two norms, with
a learned gate for every column onto the residual:

    x = scale table[ids],  h = norm(x)
    x = x + gate norm(block(h)),  h = the next block's norm(x)

Its ``backward`` gives the table's, the norms', the gates' and the adapters'
gradients, its ``step`` keeps keys and values in 8 bits. Run it on the GPU:

    python examples/voiced_text.py [--tokens 8192] [--voices 24] [--steps 20]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from brosoundml_amd import native, tokens  # noqa: E402


class TextBlock:
    """One block of `width` columns in heads of `head`, with adapters of `rank` for `voices` voices."""

    def __init__(self, ctx, width, head, voices, rank, *, causal=False, p=0.1, dtype=torch.bfloat16, seed=0):
        self.ctx, self.width, self.heads, self.head, self.causal, self.p = ctx, width, width // head, head, causal, p
        g = torch.Generator().manual_seed(seed)

        def t(*shape, by, ty=dtype):
            return (torch.randn(*shape, generator=g) * by).to(ty).cuda()

        def ints(*v):
            return torch.tensor(v, dtype=torch.int32, device="cuda")

        self.wqkv, self.wo = t(3 * width, width, by=width ** -0.5), t(width, width, by=width ** -0.5)
        self.bo = t(width, by=0.02)
        self.scale = torch.full((voices,), 1.0, device="cuda")
        # masters in float, the copies that the kernels read in `dtype`
        self.master = [t(voices, 3 * rank, width, by=width ** -0.5, ty=torch.float32),
                       torch.zeros(voices, 3 * width, rank, device="cuda"),
                       t(voices, rank, width, by=width ** -0.5, ty=torch.float32),
                       torch.zeros(voices, width, rank, device="cuda")]
        self.low = [m.to(dtype) for m in self.master]
        self.units = ints(0, width, 2 * width, 3 * width), ints(0, width)

    def _qkv(self, x, voice, **kw):
        return tokens.adapter_proj(self.ctx, x, self.wqkv, *self.low[:2], self.scale, voice, self.units[0], **kw)

    def _split(self, qkv):
        """The queries, keys and values of fused rows, as (rows, heads, head) views."""
        return qkv.view(qkv.shape[0], 3, self.heads, self.head).unbind(1)

    def mix(self, x, voice, offsets, seed, step):
        """What the block adds to its input before dropout, and what ``mix_backward`` takes."""
        drop = (self.p, seed, 3 * step)
        qkv, h1 = self._qkv(x, voice, drop=drop, keep_h=True)
        q, k, v = self._split(qkv)
        o, lse = tokens.attention(self.ctx, q, k, v, offsets, causal=self.causal)
        z, h2 = tokens.adapter_proj(self.ctx, o.reshape(x.shape), self.wo, *self.low[2:], self.scale, voice, self.units[1],
                                    bias=self.bo, drop=(self.p, seed, 3 * step + 1), keep_h=True)
        return z, (x, voice, offsets, qkv, h1, o, lse, h2, seed, step)

    def mix_backward(self, dz, kept):
        """dx of ``mix`` and the adapters' gradients (float), in the order of ``master``."""
        x, voice, offsets, qkv, h1, o, lse, h2, seed, step = kept
        do, da2, db2 = tokens.adapter_proj_bwd(self.ctx, o.view(x.shape), self.wo, *self.low[2:], self.scale, voice,
                                               self.units[1], h2, dz, drop=(self.p, seed, 3 * step + 1))
        dqkv = torch.empty_like(qkv)
        dq, dk, dv = self._split(dqkv)
        tokens.attention_bwd(self.ctx, *self._split(qkv), o, lse, do.view(o.shape), offsets, causal=self.causal,
                             dq=dq, dk=dk, dv=dv)
        dx, da1, db1 = tokens.adapter_proj_bwd(self.ctx, x, self.wqkv, *self.low[:2], self.scale, voice, self.units[0],
                                               h1, dqkv, drop=(self.p, seed, 3 * step))
        return dx, (da1, db1, da2, db2)

    def forward(self, x, voice, offsets, seed, step):
        """y and what ``backward`` takes. Dropout masks are the seed's and the step's, nothing of them is stored."""
        z, kept = self.mix(x, voice, offsets, seed, step)
        return tokens.dropout(self.ctx, z, self.p, seed, 3 * step + 2, residual=x), kept

    def backward(self, dy, kept):
        """dx and the adapters' gradients (float), in the order of ``master``."""
        seed, step = kept[-2:]
        dx, grads = self.mix_backward(tokens.dropout(self.ctx, dy, self.p, seed, 3 * step + 2), kept)
        return dy + dx, grads

    def update(self, grads, rate):
        for m, l, g in zip(self.master, self.low, grads):
            m.sub_(g, alpha=rate)
            l.copy_(m)

    def step(self, x, voice, cache, filled, slot):
        """One new token (x: a row per utterance) over the (utterances * slot, 2, heads, head) cache, of which
        ``filled`` holds how many tokens of every slot there are, fewer than `slot`; they become one more."""
        n = x.shape[0]
        q, k, v = self._split(self._qkv(x, voice))
        at = torch.arange(n, device=x.device) * slot + filled
        cache[at, 0], cache[at, 1] = k, v
        filled += 1
        rows = torch.arange(n + 1, dtype=torch.int32, device=x.device)
        o, _ = tokens.attention(self.ctx, q, cache[:, 0], cache[:, 1], rows, rows * slot, filled, causal=True)
        z = tokens.adapter_proj(self.ctx, o.reshape(n, self.width), self.wo, *self.low[2:], self.scale, voice,
                                self.units[1], bias=self.bo)
        return x + z


class TextModel:
    """`layers` TextBlocks over a table of `vocab` rows, each block between two norms (`kind`) and behind a gate."""

    def __init__(self, ctx, vocab, width, head, voices, rank, *, layers=2, kind="layer", causal=False, p=0.0, dtype=torch.bfloat16, seed=0):
        self.ctx, self.kind, self.scale = ctx, kind, width ** 0.5
        self.blocks = [TextBlock(ctx, width, head, voices, rank, causal=causal, p=p, dtype=dtype, seed=seed + i) for i in range(layers)]
        g = torch.Generator().manual_seed(seed + 99)

        def t(*shape, mid=0.0, by=0.1):
            return (mid + torch.randn(*shape, generator=g) * by).to(dtype).cuda()

        self.table = t(vocab, width, by=width ** -0.5)
        self.pre = [(t(width, mid=1.0), t(width) if kind == "layer" else None) for _ in range(layers + 1)]  # the last is the output's
        self.post = [(t(width, mid=1.0), None) for _ in range(layers)]
        self.gate = [t(width, mid=0.5) for _ in range(layers)]

    def _rule(self, i):
        """What stands behind block i: its norm and gate, and the next one's norm."""
        return dict(post=self.post[i], gate=self.gate[i], pre=self.pre[i + 1], kind=self.kind)

    def forward(self, ids, voice, offsets, seed, step):
        """The normed output rows, and what ``backward`` takes."""
        x = tokens.embedding(self.ctx, self.table, ids, scale=self.scale)
        _, h, first = tokens.residual_norm(self.ctx, x, pre=self.pre[0], kind=self.kind, keep=True)
        kept = []
        for i, block in enumerate(self.blocks):
            z, inner = block.mix(h, voice, offsets, seed, step * len(self.blocks) + i)
            r, h, stats = tokens.residual_norm(self.ctx, x, z, keep=True, **self._rule(i))
            kept.append((x, z, stats, inner))
            x = r
        return h, (ids, first, kept)

    def backward(self, dh, state):
        """The gradients: "table", "first" (the first norm's weight and bias), and of every block "gate", "post",
        "pre" (the next norm's) and "adapters"; all but the tensors in between are float."""
        ids, first, kept = state
        dx, blocks = None, []
        for i in reversed(range(len(kept))):
            x, z, stats, inner = kept[i]
            dx, dz, dgate, dpost, dpre = tokens.residual_norm_bwd(self.ctx, x, z, dx, dh, stats, **self._rule(i))
            dh, adapters = self.blocks[i].mix_backward(dz, inner)
            blocks.insert(0, {"gate": dgate, "post": dpost, "pre": dpre, "adapters": adapters})
        dx, _, _, _, dfirst = tokens.residual_norm_bwd(self.ctx, kept[0][0], None, dx, dh, first, pre=self.pre[0], kind=self.kind)
        table = tokens.embedding_bwd(self.ctx, ids, dx, self.table.shape[0], scale=self.scale)
        return {"table": table, "first": dfirst, "blocks": blocks}

    def caches(self, utterances, slot):
        """An 8-bit cache for every block, `slot` tokens for each utterance."""
        b = self.blocks[0]
        return [tokens.new_cache(self.ctx, utterances * slot, b.heads, b.head) for _ in self.blocks]

    def step(self, ids, voice, caches, filled, slot):
        """The next token of every utterance (ids: one each) over the caches, of which ``filled`` holds how many
        tokens of every slot there are, fewer than `slot`; they become one more. The new rows' normed output."""
        n = ids.shape[0]
        rows = torch.arange(n + 1, dtype=torch.int32, device=ids.device)
        where = rows, rows * slot, filled.add_(1)
        x = tokens.embedding(self.ctx, self.table, ids, scale=self.scale)
        _, h = tokens.residual_norm(self.ctx, x, pre=self.pre[0], kind=self.kind)
        for i, (b, cache) in enumerate(zip(self.blocks, caches)):
            q, k, v = b._split(b._qkv(h, voice))
            tokens.cache_write(self.ctx, k, v, cache, *where)
            o, _ = tokens.cache_attention(self.ctx, q, cache, *where, causal=True)
            z = tokens.adapter_proj(self.ctx, o.reshape(n, b.width), b.wo, *b.low[2:], b.scale, voice, b.units[1], bias=b.bo)
            x, h = tokens.residual_norm(self.ctx, x, z, **self._rule(i))
        return h


def utterances(total, voices, seed=0):
    """Offsets of utterances of 20 to 510 tokens that make `total`, and every token's voice."""
    g = torch.Generator().manual_seed(seed)
    cuts = [0]
    while cuts[-1] < total:
        cuts.append(min(total, cuts[-1] + int(torch.randint(20, 511, (1,), generator=g))))
    who = torch.randint(0, voices, (len(cuts) - 1,), generator=g)
    voice = torch.repeat_interleave(who, torch.tensor(cuts).diff()).int()
    return torch.tensor(cuts, dtype=torch.int32).cuda(), voice.cuda()


def train(ctx, *, tokens_=8192, width=1024, head=64, voices=24, rank=16, steps=20, rate=2.0, dtype=torch.bfloat16, seed=0):
    """Fits the voices' adapters to targets that another set of adapters made; the mean squared errors by step."""
    p = 0.05
    block, teacher = (TextBlock(ctx, width, head, voices, rank, p=q, dtype=dtype, seed=seed) for q in (p, 0.0))
    g = torch.Generator().manual_seed(seed + 1)
    teacher.low[1].copy_(torch.randn(teacher.low[1].shape, generator=g) * 0.1)
    teacher.low[3].copy_(torch.randn(teacher.low[3].shape, generator=g) * 0.1)
    offsets, voice = utterances(tokens_, voices, seed)
    x = torch.randn(tokens_, width, generator=g).to(dtype).cuda()
    target, _ = teacher.forward(x, voice, offsets, 0, 0)
    losses = []
    for i in range(steps):
        y, kept = block.forward(x, voice, offsets, seed + 7, i)
        diff = y.float() - target.float()
        losses.append(diff.square().mean())
        _, grads = block.backward((diff * (2.0 / tokens_)).to(dtype), kept)
        block.update(grads, rate)
    return [float(v) for v in losses], block


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=8192)
    ap.add_argument("--voices", type=int, default=24)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    ctx = native.Context(0)
    train(ctx, tokens_=a.tokens, voices=a.voices, steps=1)
    torch.cuda.synchronize()
    t = time.perf_counter()
    losses, block = train(ctx, tokens_=a.tokens, voices=a.voices, steps=a.steps)
    torch.cuda.synchronize()
    print(f"{a.steps} steps of {a.tokens} tokens in {a.voices} voices: {time.perf_counter() - t:.3f} s with the data's making")
    print("mean squared error by step:", " ".join(f"{v:.4f}" for v in losses[::max(1, a.steps // 10)]), f"... {losses[-1]:.4f}")
    # one token at a time, every voice its own utterance
    slot, n = 512, a.voices
    cache = torch.zeros(n * slot, 2, block.heads, block.head, dtype=torch.bfloat16, device="cuda")
    filled = torch.zeros(n, dtype=torch.int32, device="cuda")
    x, voice = torch.randn(n, block.width, device="cuda").bfloat16(), torch.arange(n, dtype=torch.int32, device="cuda")
    for i in range(64):
        x = torch.nn.functional.normalize(block.step(x, voice, cache, filled, slot).float(), dim=1).mul(block.width ** 0.5).bfloat16()
    torch.cuda.synchronize()
    print(f"64 tokens for {n} utterances, finite: {bool(torch.isfinite(x).all())}")
    # the same from token ids on, through a stack of blocks over 8-bit caches
    model = TextModel(ctx, 181, 1024, 64, n, 16)
    caches, filled = model.caches(n, slot), torch.zeros(n, dtype=torch.int32, device="cuda")
    ids = torch.arange(n, dtype=torch.int32, device="cuda")
    for _ in range(64):
        ids = (model.step(ids, voice, caches, filled, slot).float() @ model.table.float().t()).argmax(1).int()
    print(f"64 tokens for {n} utterances over 8-bit caches:", ids.tolist()[:8])
    off, voice = utterances(a.tokens, n)
    h, state = model.forward(torch.randint(0, 181, (a.tokens,)).int().cuda(), voice, off, 1, 0)
    grads = model.backward(torch.randn_like(h) * 1e-3, state)
    print(f"{a.tokens} tokens through {len(model.blocks)} blocks and back, the table's gradient:", tuple(grads["table"].shape))


if __name__ == "__main__":
    main()
