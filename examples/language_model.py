"""The operators of matrix_b200.lm as a language model uses them: training steps of a small decoder with hand-
written backward passes, a decode loop that chooses tokens under penalties and a grammar mask, and the same model served:
prompts of different lengths packed into one pass, then a token at a time for all of them over a paged cache.

The matrix products of the weights are torch's; every other pass over the activations is this framework's: the norms
around a block with its gate, dropout and residual, the norms of the heads and their rotary positions, dropout, the softmax
over the scores, the cache and the attention over it, the rules on the logits and the ArgMax that chooses.  Run it with

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
    logits from the embedding's transpose.  head_norm: queries and keys are normed for each head before they are turned.
    All parameters float32."""

    def __init__(self, vocab=256, width=64, heads=4, kv_heads=2, hidden=128, p=0.1, seed=0, device="cuda", head_norm=False):
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
        self.head_norm = head_norm
        if head_norm:
            self.w |= {"q_norm": torch.ones(self.head, device=device), "k_norm": torch.ones(self.head, device=device)}
        self.frequencies, self.scale = lm.rotary_frequencies(self.head, device=device)

    def split(self, qkv):
        q, k, v = qkv.split([self.heads * self.head, self.kv_heads * self.head, self.kv_heads * self.head], -1)
        shape = (*qkv.shape[:-1], -1, self.head)
        return q.reshape(shape), k.reshape(shape), v.reshape(shape)

    def turn(self, q, k, positions, save=False):
        """Queries and keys normed, if the model does, and turned: (q, k, what the backward pass needs)."""
        if not self.head_norm:
            return *lm.rotary(q, k, positions, self.frequencies, scale=self.scale), None
        o = lm.head_norm_rotary(q, k, positions, self.frequencies, q_weight=self.w["q_norm"], k_weight=self.w["k_norm"],
                                scale=self.scale, save_rstd=save)
        return o.q, o.k, (q, k, o.q_rstd, o.k_rstd)

    def turn_backward(self, d_q, d_k, positions, saved, g):
        """The gradients at turn's inputs; those of its weights go into g."""
        if not self.head_norm:
            return lm.rotary(d_q, d_k, positions, self.frequencies, scale=self.scale, inverse=True)
        q, k, q_rstd, k_rstd = saved
        d = lm.head_norm_rotary_backward(d_q, d_k, q, k, positions, self.frequencies, q_rstd=q_rstd, k_rstd=k_rstd,
                                         q_weight=self.w["q_norm"], k_weight=self.w["k_norm"], scale=self.scale)
        g["q_norm"], g["k_norm"] = d.q_weight, d.k_weight
        return d.q, d.k

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
        q, k, saved = self.turn(q, k, positions, save=True)
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
        d_q, d_k = self.turn_backward(d_q, d_k, positions, saved, g)
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
            q, k, _ = self.turn(q, k, torch.full((1,), t, dtype=torch.int32, device=dev))
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


    def attend(self, x, positions, cache, slots, attention):
        """One pass of tokens [tokens, width] through the model: their keys and values go to the cache's slots, and
        attention(q, k, v) is what their queries see.  Returns the last norm's output."""
        w = self.w
        a = lm.block_norm(x, next_weight=w["norm0"], save_rstd=False)
        q, k, v = self.split(a.normed @ w["qkv"])
        q, k, _ = self.turn(q, k, positions)
        lm.cache_write(cache, k, v, slots)
        mixed = attention(q, k, v).flatten(1)
        a = lm.block_norm(x, mixed @ w["out"], post_weight=w["post1"], gate=w["gate1"], next_weight=w["norm1"], save_rstd=False)
        return lm.block_norm(a.residual, (a.normed @ w["up"]).relu() @ w["down"], post_weight=w["post2"], gate=w["gate2"],
                             next_weight=w["norm2"], save_rstd=False).normed

    def generate(self, prompts: list, count: int, cache_dtype=torch.float32, page=8, prefix=0) -> tuple:
        """`count` tokens more for each of prompts (token tensors of any lengths), all at once: the prompts packed into one
        pass, then one pass a token over a paged cache.  The first `prefix` tokens of each prompt (fewer than it has) make a
        pass of their own, and the rest of the prompt reads their keys and values back from the cache.  Returns the tokens
        [prompts, count] and the logits that chose them [prompts, count, vocab]."""
        w, dev, n = self.w, prompts[0].device, len(prompts)
        lengths = [len(t) for t in prompts]
        pages = -(-(max(lengths) + count) // page)
        table = torch.randperm(n * pages, device=dev).to(torch.int32).view(n, pages)  # in any order
        cache = lm.kv_cache(n * pages, page, self.kv_heads, self.head, cache_dtype, device=dev)

        def slots(sequence, position):
            return table[sequence, position // page] * page + position % page

        def starts(values):
            return torch.tensor([0, *values], device=dev).cumsum(0).to(torch.int32)

        def prompt_pass(first, last):  # tokens first[i] .. last[i] - 1 of prompt i
            tokens = torch.cat([t[a:b] for t, a, b in zip(prompts, first, last)])
            at = torch.cat([torch.arange(a, b, device=dev) for a, b in zip(first, last)])
            of = torch.cat([torch.full((b - a,), i, device=dev) for i, (a, b) in enumerate(zip(first, last))])
            every = torch.cat([slots(i, torch.arange(b, device=dev)) for i, b in enumerate(last)])

            def attention(q, k, v):
                if any(first):  # what came before is in the cache
                    k, v = lm.cache_read(cache, every, dtype=q.dtype)
                return lm.prompt_attention(q, k, v, starts([b - a for a, b in zip(first, last)]), k_starts=starts(last))

            return self.attend(w["embed"][tokens], at, cache, slots(of, at), attention)

        if prefix:
            prompt_pass([0] * n, [prefix] * n)
        hidden = prompt_pass([prefix] * n, lengths)
        hidden = hidden[starts([m - prefix for m in lengths])[1:].long() - 1]  # of each prompt's last token
        tokens, chosen = torch.empty(n, count, dtype=torch.int32, device=dev), []
        sequence, length = torch.arange(n, device=dev), torch.tensor(lengths, dtype=torch.int32, device=dev)
        for step in range(count):
            logits = hidden @ w["embed"].mT
            chosen.append(logits)
            tokens[:, step] = backend.reduce("argmax", logits, 1)
            if step + 1 < count:
                at = length + step
                hidden = self.attend(w["embed"][tokens[:, step].long()], at, cache, slots(sequence, at),
                                     lambda q, k, v: lm.decode_attention(q, cache, table, at + 1))
        return tokens, torch.stack(chosen, 1)


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
    print(model.generate([cycle[0, :6], cycle[1, :11], cycle[2, :3]], 10)[0].tolist())


if __name__ == "__main__":
    main()
