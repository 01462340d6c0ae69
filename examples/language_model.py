"""The row operators of matrix_b200.lm as a language model uses them: training steps of a small decoder with hand-
written backward passes, and a decode loop that chooses tokens under penalties and a grammar mask.

The matrix products are torch's; every other pass over the activations is this framework's: the norms around a block
with its gate, dropout and residual, rotary positions, dropout, the softmax over the scores, the rules on the logits and
the ArgMax that chooses.  Run it with

    python examples/language_model.py
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from matrix_b200 import backend, lm

LOWEST = torch.finfo(torch.float32).min


def softmax(x: torch.Tensor) -> torch.Tensor:
    return backend.softmax_lastdim(x.contiguous())


class Decoder:
    """Embedding, one attention block, one feed-forward block (each between two norms, with a gate per channel), and
    logits from the embedding's transpose.  All parameters float32."""

    def __init__(self, vocab=256, width=64, heads=4, kv_heads=2, hidden=128, p=0.1, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)

        def normal(*shape, std):
            return (torch.randn(*shape, generator=g) * std).to(device)

        self.heads, self.kv_heads, self.head, self.p = heads, kv_heads, width // heads, p
        self.w = {
            "embed": normal(vocab, width, std=0.5), "qkv": normal(width, (heads + 2 * kv_heads) * self.head, std=0.1),
            "out": normal(width, width, std=0.1), "up": normal(width, hidden, std=0.1), "down": normal(hidden, width, std=0.1),
            "norm0": torch.ones(width, device=device), "post1": torch.ones(width, device=device),
            "gate1": torch.full((width,), 0.5, device=device), "norm1": torch.ones(width, device=device),
            "post2": torch.ones(width, device=device), "gate2": torch.full((width,), 0.5, device=device),
            "norm2": torch.ones(width, device=device)}
        self.frequencies, self.scale = lm.rotary_frequencies(self.head, device=device)

    def split(self, qkv):
        q, k, v = qkv.split([self.heads * self.head, self.kv_heads * self.head, self.kv_heads * self.head], -1)
        shape = (*qkv.shape[:-1], -1, self.head)
        return q.reshape(shape), k.reshape(shape), v.reshape(shape)

    # -- training ----------------------------------------------------------------------------
    def step(self, tokens: torch.Tensor, seed: int):
        """Loss and parameter gradients for next-token prediction on tokens [batch, length] (length - 1 a multiple of
        4).  Each dropout of the step has an offset of its own; the backward pass names the same ones."""
        w, p = self.w, self.p
        inputs, targets = tokens[:, :-1], tokens[:, 1:]
        batch, n = inputs.shape
        positions = torch.arange(n, dtype=torch.int32, device=tokens.device)
        x0 = w["embed"][inputs]
        a0 = lm.block_norm(x0, next_weight=w["norm0"])

        q, k, v = self.split(a0.normed @ w["qkv"])
        q, k = lm.rotary(q, k, positions, self.frequencies, scale=self.scale)
        group = self.heads // self.kv_heads
        qh, kh, vh = q.transpose(1, 2), *(t.repeat_interleave(group, 2).transpose(1, 2) for t in (k, v))
        causal = torch.ones(n, n, dtype=torch.bool, device=tokens.device).tril()
        scores = torch.where(causal, qh @ kh.mT / self.head ** 0.5, LOWEST)
        probs = softmax(scores)
        mixed = (probs @ vh).transpose(1, 2).reshape(batch, n, -1)
        how1 = dict(post_weight=w["post1"], gate=w["gate1"], next_weight=w["norm1"], dropout=p, seed=seed, offset=1)
        b1 = mixed @ w["out"]
        a1 = lm.block_norm(x0, b1, **how1)

        up = a1.normed @ w["up"]
        act = lm.dropout(up.relu(), p, seed, 2)
        how2 = dict(post_weight=w["post2"], gate=w["gate2"], next_weight=w["norm2"], dropout=p, seed=seed, offset=3)
        b2 = act @ w["down"]
        a2 = lm.block_norm(a1.residual, b2, **how2)

        logits = a2.normed @ w["embed"].mT
        prob = softmax(logits.view(-1, logits.shape[-1])).view_as(logits)
        chosen = prob.gather(2, targets[..., None])
        loss = -chosen.log().mean()

        # backward, in the opposite order
        g = {}
        d_logits = prob.scatter_add(2, targets[..., None], torch.full_like(chosen, -1.0)) / targets.numel()
        g["embed"] = torch.einsum("bnv,bnd->vd", d_logits, a2.normed)
        d2 = lm.block_norm_backward(None, d_logits @ w["embed"], a2.residual, b2, post_rstd=a2.post_rstd,
                                    next_rstd=a2.next_rstd, **how2)
        g["post2"], g["gate2"], g["norm2"] = d2.post_weight, d2.gate, d2.next_weight
        g["down"] = torch.einsum("bnh,bnd->hd", act, d2.branch)
        d_up = lm.dropout(d2.branch @ w["down"].mT, p, seed, 2) * (up > 0)
        g["up"] = torch.einsum("bnd,bnh->dh", a1.normed, d_up)
        d1 = lm.block_norm_backward(d2.residual, d_up @ w["up"].mT, a1.residual, b1, post_rstd=a1.post_rstd,
                                    next_rstd=a1.next_rstd, **how1)
        g["post1"], g["gate1"], g["norm1"] = d1.post_weight, d1.gate, d1.next_weight
        g["out"] = torch.einsum("bnc,bnd->cd", mixed, d1.branch)
        d_mixed = (d1.branch @ w["out"].mT).view(batch, n, self.heads, self.head).transpose(1, 2)
        d_probs = d_mixed @ vh.mT
        d_scores = probs * (d_probs - (d_probs * probs).sum(-1, keepdim=True)) / self.head ** 0.5
        shared = (batch, n, self.kv_heads, group, self.head)
        d_q = (d_scores @ kh).transpose(1, 2).contiguous()
        d_k = (d_scores.mT @ qh).transpose(1, 2).reshape(shared).sum(3)
        d_v = (probs.mT @ d_mixed).transpose(1, 2).reshape(shared).sum(3)
        d_q, d_k = lm.rotary(d_q, d_k, positions, self.frequencies, scale=self.scale, inverse=True)
        d_qkv = torch.cat([t.flatten(2) for t in (d_q, d_k, d_v)], -1)
        g["qkv"] = torch.einsum("bnd,bnc->dc", a0.normed, d_qkv)
        d0 = lm.block_norm_backward(d1.residual, d_qkv @ w["qkv"].mT, x0, next_rstd=a0.next_rstd, next_weight=w["norm0"])
        g["norm0"] = d0.next_weight
        g["embed"].index_put_((inputs,), d0.residual, accumulate=True)
        return loss, g

    # -- serving -----------------------------------------------------------------------------
    def decode(self, prompt: torch.Tensor, count: int, repetition=1.3, frequency=0.2, presence=0.1, bias=None,
               allowed: torch.Tensor | None = None) -> torch.Tensor:
        """`count` more tokens for each of prompt [batch, length], one at a time over a cache of keys and values:
        the most likely token after the rules on the logits.  bias: {token: value}; allowed: the mask's words."""
        w, dev = self.w, prompt.device
        batch, length = prompt.shape
        total = (length + count + 3) // 4 * 4  # rows of the softmax are multiples of 4
        keys = torch.zeros(batch, self.heads, total, self.head, device=dev)
        values = torch.zeros_like(keys)
        tokens = torch.full((batch, length + count), -1, dtype=torch.int32, device=dev)
        tokens[:, :length] = prompt
        rows = torch.ones(batch, device=dev)
        rules = dict(repetition=rows * repetition, frequency=rows * frequency, presence=rows * presence, mask=allowed,
                     prompt_lengths=torch.full((batch,), length, dtype=torch.int32, device=dev))
        if bias:
            rules |= dict(bias_tokens=torch.tensor(list(bias), dtype=torch.int32, device=dev),
                          bias_values=torch.tensor(list(bias.values()), dtype=torch.float32, device=dev))
        group = self.heads // self.kv_heads
        for t in range(length + count - 1):
            x = w["embed"][tokens[:, t].long()][:, None]  # [batch, 1, width]
            a = lm.block_norm(x, next_weight=w["norm0"], save_rstd=False)
            q, k, v = self.split(a.normed @ w["qkv"])
            at = torch.full((1,), t, dtype=torch.int32, device=dev)
            lm.rotary(q, k, at, self.frequencies, scale=self.scale, out=(q, k))
            keys[:, :, t] = k[:, 0].repeat_interleave(group, 1)
            values[:, :, t] = v[:, 0].repeat_interleave(group, 1)
            scores = (q.transpose(1, 2) @ keys.mT / self.head ** 0.5)[:, :, 0]
            scores[:, :, t + 1:] = LOWEST
            mixed = (softmax(scores)[:, :, None] @ values).transpose(1, 2).reshape(batch, 1, -1)
            a = lm.block_norm(x, mixed @ w["out"], post_weight=w["post1"], gate=w["gate1"], next_weight=w["norm1"],
                              save_rstd=False)
            a = lm.block_norm(a.residual, (a.normed @ w["up"]).relu() @ w["down"], post_weight=w["post2"], gate=w["gate2"],
                              next_weight=w["norm2"], save_rstd=False)
            if t + 1 < length:
                continue
            logits = (a.normed @ w["embed"].mT)[:, 0]
            lengths = torch.full((batch,), t + 1, dtype=torch.int32, device=dev)
            lm.logits_rules(logits, tokens=tokens, lengths=lengths, **rules, out=logits)
            tokens[:, t + 1] = backend.reduce("argmax", logits, 1)
        return tokens[:, length:]


def main() -> None:
    torch.cuda.set_device(0)
    backend.init(0)
    model = Decoder()
    cycle = torch.arange(17 * 8, device="cuda").view(8, 17) * 3 % 64  # tokens that count in threes
    for i in range(60):
        loss, gradients = model.step(cycle, seed=i)
        for name, g in gradients.items():
            model.w[name] -= 0.5 * g
        if i % 20 == 0 or i == 59:
            print(f"step {i:3d}  loss {loss.item():.4f}")
    mask = torch.zeros(8, dtype=torch.int32, device="cuda")
    mask[:2] = -1  # a grammar that allows tokens 0 .. 63
    print(model.decode(cycle[:2, :6], 10, repetition=1.0, frequency=0.0, presence=0.0, allowed=mask).tolist())


if __name__ == "__main__":
    main()
