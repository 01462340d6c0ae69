"""The attention operators together, as examples/language_model.py uses them: a model with normed heads trained, and served
over a paged cache (prompts of different lengths in one pass, a prefix read back, then a token at a time), against the same
model in 64 bits."""
import importlib.util

import pytest
import torch

from tests import attention_reference as att
from tests.conftest import REPO
from tests.test_gpu_lm_example import rotate, unit

pytestmark = pytest.mark.gpu


@pytest.fixture
def example(gpu):
    spec = importlib.util.spec_from_file_location("language_model", REPO / "examples" / "language_model.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain(model, w, tokens, mask=None, quantised=False):
    """The decoder's logits in 64 bits for tokens [batch, length]; quantised: keys and values as a cache in 8 bits holds
    them."""
    mask = mask or (lambda shape, offset: 1.0)
    batch, n = tokens.shape
    x = w["embed"][tokens]
    q, k, v = model.split(unit(x) * w["norm0"] @ w["qkv"])
    if model.head_norm:
        q, k = unit(q) * w["q_norm"], unit(k) * w["k_norm"]
    positions, f = torch.arange(n).expand(batch, n), model.frequencies.cpu()
    q, k = (torch.stack([rotate(t[..., i, :], positions, f) for i in range(t.shape[-2])], -2) for t in (q, k))
    if quantised:
        k, v = att.quantise(k)[0], att.quantise(v)[0]
    group = model.heads // model.kv_heads
    q, k, v = q.transpose(1, 2), *(t.repeat_interleave(group, 2).transpose(1, 2) for t in (k, v))
    scores = (q @ k.mT / model.head ** 0.5).masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -torch.inf)
    mixed = (scores.softmax(-1) @ v).transpose(1, 2).reshape(batch, n, -1)
    b = unit(mixed @ w["out"]) * w["post1"]
    x = x + w["gate1"] * b * mask(b.shape, 1)
    h = (unit(x) * w["norm1"] @ w["up"]).relu()
    b = unit(h * mask(h.shape, 2) @ w["down"]) * w["post2"]
    x = x + w["gate2"] * b * mask(b.shape, 3)
    return unit(x) * w["norm2"] @ w["embed"].mT


def test_gradients_with_normed_heads(example):
    """The bounds are those of the model without them: float32 against 64 bits through about a dozen products."""
    from tests import lm_reference as ref

    model = example.Decoder(seed=4, head_norm=True)
    for name in ("q_norm", "k_norm"):
        model.w[name] += 0.3 * torch.randn(model.head, generator=torch.Generator().manual_seed(7)).cuda()
    tokens = torch.randint(0, 256, (2, 13), generator=torch.Generator().manual_seed(1))
    loss, got = model.step(tokens.cuda(), seed=99)
    w = {k: v.cpu().double().requires_grad_() for k, v in model.w.items()}

    def mask(shape, offset):
        return ref.keep_mask(model.p, 99, offset, shape[0] * shape[1], shape[2]).view(shape)

    want = torch.nn.functional.cross_entropy(plain(model, w, tokens[:, :-1], mask).flatten(0, 1), tokens[:, 1:].flatten())
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    assert got.keys() == w.keys()
    for name, g in got.items():
        exact = w[name].grad
        assert (g.cpu().double() - exact).norm() <= 1e-4 * exact.norm(), name


@pytest.mark.parametrize("head_norm", [False, True])
@pytest.mark.parametrize("prefix", [0, 2])
def test_serving_follows_the_model(example, head_norm, prefix):
    """Logits in float32 through about a dozen products of at most 256 terms of order 1: 1e-4 of their size, as the training
    step's gradients; a token is the most likely one of the logits that it is returned with."""
    model = example.Decoder(seed=5, head_norm=head_norm)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 256, (n,), generator=g) for n in (7, 3, 29, 12)]
    tokens, logits = model.generate([t.cuda() for t in prompts], 9, page=4, prefix=prefix)
    w = {k: v.cpu().double() for k, v in model.w.items()}
    assert torch.equal(tokens.long(), logits.argmax(-1))
    for i, prompt in enumerate(prompts):
        full = torch.cat([prompt, tokens[i].cpu().long()])[None]
        want = plain(model, w, full)[0, len(prompt) - 1:-1]
        assert (logits[i].cpu().double() - want).abs().max() <= 1e-4 * want.abs().max(), i


def test_serving_over_8_bits(example):
    """The same with the cache in 8 bits: against the model whose keys and values are rounded to them -- for the prompts'
    own pass, which does not read them back, nothing is.  A key within 2^-20 of a border between two bytes may go either
    way and move a logit by 2^-4 of its share: the bound allows for one such element a step."""
    model = example.Decoder(seed=6)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 256, (n,), generator=g) for n in (9, 17)]
    tokens, logits = model.generate([t.cuda() for t in prompts], 4, cache_dtype=torch.float8_e4m3fn, page=8)
    exact, _ = model.generate([t.cuda() for t in prompts], 4, page=8)
    w = {k: v.cpu().double() for k, v in model.w.items()}
    for i, prompt in enumerate(prompts):
        want = plain(model, w, prompt[None])[0, -1]
        assert (logits[i, 0].cpu().double() - want).abs().max() <= 1e-4 * want.abs().max()
        full = torch.cat([prompt, tokens[i].cpu().long()])[None]
        want = plain(model, w, full, quantised=True)[0, len(prompt):-1]
        assert (logits[i, 1:].cpu().double() - want).abs().max() <= 2e-2 * want.abs().max(), i
    assert torch.equal(tokens[:, 0], exact[:, 0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["plain", "8 bits"])
def test_a_prompt_in_pieces(gpu, dtype, kind):
    """Half types through the operators in turn: norms and rotation, the cache, a prompt's second half over its first read
    back, then a token over the same cache: equal to the formulas over what the cache holds."""
    from matrix_b200 import lm

    n, cut, qh, kh, head, page = 300, 130, 8, 2, 128, 16
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, head, generator=g).to(dtype).cuda() for h in (qh, kh, kh))
    f, scale = lm.rotary_frequencies(head)
    w = torch.ones(head, dtype=dtype, device="cuda")
    o = lm.head_norm_rotary(q, k, torch.arange(n, device="cuda"), f, q_weight=w, k_weight=w, scale=scale)
    cache = lm.kv_cache(30, page, kh, head, dtype if kind == "plain" else torch.float8_e4m3fn)
    table = torch.randperm(30, generator=g).to(torch.int32).cuda()
    at = torch.arange(n, device="cuda")
    slots = table[at // page] * page + at % page
    lm.cache_write(cache, o.k, v, slots)
    keys, values = lm.cache_read(cache, slots, dtype=dtype)
    held = [x.cpu().double() for x in (keys, values)]
    if kind == "plain":
        assert torch.equal(keys, o.k) and torch.equal(values, v)
    got = lm.prompt_attention(o.q[cut:], keys, values, torch.tensor([0, n - cut], dtype=torch.int32).cuda(),
                              k_starts=torch.tensor([0, n], dtype=torch.int32).cuda())
    q64 = o.q.cpu().double()
    want, bound = att.prompt(q64[cut:], *held, [0, n - cut], [0, n], head ** -0.5, True, dtype)
    att.assert_close(got, want, bound)
    one = lm.decode_attention(o.q[-1:], cache, table[None], torch.tensor([n], dtype=torch.int32).cuda())
    # a cache in 8 bits may hold more than the half type that it was read to
    pages, slot = (table[at // page] * page + at % page).cpu() // page, at.cpu() % page
    full = lm.cache_read(cache, slots, dtype=torch.float32 if kind != "plain" else dtype)
    k_pages, v_pages = torch.zeros(30, page, kh, head, dtype=torch.float64), torch.zeros(30, page, kh, head, dtype=torch.float64)
    k_pages[pages.long(), slot], v_pages[pages.long(), slot] = (x.cpu().double() for x in full)
    want, bound = att.decode(q64[-1:], k_pages, v_pages, table[None].cpu(), [n], head ** -0.5, dtype)
    att.assert_close(one, want, bound)
