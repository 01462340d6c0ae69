"""examples/language_model.py: the row operators together.  Its hand-written gradients against torch's autograd in 64 bits
of the same model, its decode loop against a plain one, and its command."""
import importlib.util
import subprocess
import sys

import pytest
import torch

from tests import lm_reference as ref
from tests.conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.fixture
def example(gpu):
    spec = importlib.util.spec_from_file_location("language_model", REPO / "examples" / "language_model.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def unit(x):
    return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()


def plain(model, w, tokens, mask):
    """The decoder's logits in 64 bits; mask(shape, offset): the dropout factors."""
    batch, n = tokens.shape
    x = w["embed"][tokens]
    q, k, v = model.split(unit(x) * w["norm0"] @ w["qkv"])
    positions = torch.arange(n).expand(batch, n)
    f = model.frequencies.cpu()
    turn = lambda t: torch.stack([rotate(t[..., i, :], positions, f) for i in range(t.shape[-2])], -2)  # noqa: E731
    q, k = turn(q), turn(k)
    group = model.heads // model.kv_heads
    q, k, v = q.transpose(1, 2), k.repeat_interleave(group, 2).transpose(1, 2), v.repeat_interleave(group, 2).transpose(1, 2)
    scores = (q @ k.mT / model.head ** 0.5).masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -torch.inf)
    mixed = (scores.softmax(-1) @ v).transpose(1, 2).reshape(batch, n, -1)
    b = unit(mixed @ w["out"]) * w["post1"]
    x = x + w["gate1"] * b * mask(b.shape, 1)
    h = (unit(x) * w["norm1"] @ w["up"]).relu()
    b = unit(h * mask(h.shape, 2) @ w["down"]) * w["post2"]
    x = x + w["gate2"] * b * mask(b.shape, 3)
    return unit(x) * w["norm2"] @ w["embed"].mT


def rotate(x, positions, f):
    t = positions[..., None] * f
    a, b = x[..., :len(f)], x[..., len(f):]
    return torch.cat([a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()], -1)


def test_gradients_are_those_of_the_model(example):
    """float32 against 64 bits: activations of order 1 through about ten products of at most 256 terms keep 2^-24
    relative errors below 1e-5 of each gradient's size; 1e-4 allows for the softmax's and ReLU's own conditioning."""
    model = example.Decoder(seed=3)
    tokens = torch.randint(0, 256, (2, 13), generator=torch.Generator().manual_seed(1))
    loss, got = model.step(tokens.cuda(), seed=99)
    w = {k: v.cpu().double().requires_grad_() for k, v in model.w.items()}

    def mask(shape, offset):
        return ref.keep_mask(model.p, 99, offset, shape[0] * shape[1], shape[2]).view(shape)

    logits = plain(model, w, tokens[:, :-1], mask)
    want = torch.nn.functional.cross_entropy(logits.flatten(0, 1), tokens[:, 1:].flatten())
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    assert got.keys() == w.keys()
    for name, g in got.items():
        exact = w[name].grad
        assert (g.cpu().double() - exact).norm() <= 1e-4 * exact.norm(), name


def test_decode_follows_the_rules(example):
    model = example.Decoder(seed=5)
    prompt = torch.randint(0, 256, (3, 7), generator=torch.Generator().manual_seed(2))
    words = torch.full((8,), 0x0F0F0F0F, dtype=torch.int32)
    bias = {3: 2.0, 40: -3.0, 200: 1.0}
    got = model.decode(prompt.cuda(), 6, bias=bias, allowed=words.cuda()).cpu()
    w = {k: v.cpu().double() for k, v in model.w.items()}
    tokens = prompt.clone()
    for step in range(6):
        logits = plain(model, w, tokens, lambda shape, offset: 1.0)[:, -1]
        n = tokens.shape[1]
        ruled, _ = ref.logits_rules(logits, tokens=tokens.tolist(), lengths=[n] * 3, prompt_lengths=[7] * 3,
                                    repetition=[1.3] * 3, frequency=[0.2] * 3, presence=[0.1] * 3,
                                    bias_tokens=[list(bias)] * 3, bias_values=[list(bias.values())] * 3,
                                    mask=[words.tolist()] * 3)
        best = ruled.topk(2, 1)
        sure = best.values[:, 0] - best.values[:, 1] > 1e-4  # nearer ones may go either way in 32 bits
        assert torch.equal(got[sure, step].long(), best.indices[sure, 0])
        assert all(words[t // 32] >> (t % 32) & 1 for t in got[:, step].tolist())
        tokens = torch.cat([tokens, got[:, step:step + 1].long()], 1)


def test_command(gpu):
    out = subprocess.run([sys.executable, str(REPO / "examples" / "language_model.py")], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    losses = [float(line.split()[-1]) for line in out.stdout.splitlines() if line.startswith("step")]
    assert losses[-1] < 0.5 * losses[0]
