"""examples/speculative_decode.py: every generated token is the choice of a
dense fp32 evaluation of the same weights, drafted or not, and drafting takes
fewer steps.

A choice counts when its dense logit is within 64 u max|logit| of the largest
(u the element type's unit roundoff: the two layers round activations about
a dozen times each, and a near tie may go either way), and nine in ten have to
be the dense choice itself.
"""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")

from akili_bench_b200 import ops  # noqa: E402
import serving_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "speculative_decode.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("speculative_decode", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def dense_logits(m, w, tokens):
    f = lambda t: t.float()  # noqa: E731
    norm = lambda y: y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)  # noqa: E731
    n = len(tokens)
    table = ops.rope_table(m.MAX_POSITIONS, m.HEAD_DIM)[:n]
    c, s = table[:, None, :m.HEAD_DIM // 2], table[:, None, m.HEAD_DIM // 2:]

    def turn(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    x = f(w["embed"])[torch.tensor(tokens, device="cuda")]
    hide = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
    for layer in w["layers"]:
        qkv = (norm(x) @ f(layer["qkv"])).view(n, -1, m.HEAD_DIM)
        q, k, v = qkv.split([m.Q_HEADS, m.KV_HEADS, m.KV_HEADS], 1)
        q, k = turn(q), turn(k)
        k, v = (t.repeat_interleave(m.Q_HEADS // m.KV_HEADS, 1) for t in (k, v))
        a = torch.einsum("nhd,mhd->hnm", q, k) * m.HEAD_DIM ** -0.5
        o = torch.einsum("hnm,mhd->nhd", a.masked_fill(hide, float("-inf")).softmax(-1), v)
        x = x + o.flatten(1) @ f(layer["o"])
        y = norm(x)
        x = x + (torch.nn.functional.silu(y @ f(layer["gate"])) * (y @ f(layer["up"]))) @ f(layer["down"])
    return norm(x) @ f(w["head"])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_speculative_decode_takes_the_models_tokens(example, dtype):
    ops.device_status()
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, example.VOCAB, (n,), generator=g).tolist() for n in (61, 4, 133, 1)]
    new = 40
    drafted, steps = example.generate(prompts, new, dtype)
    plain, plain_steps = example.generate(prompts, new, dtype, drafted=False)
    assert ops.device_status() == 0
    assert plain_steps == new - 1 and steps < plain_steps
    w = example.weights(dtype)
    for seqs in (drafted, plain):
        same = total = 0
        for p, s in zip(prompts, seqs):
            assert len(s) == len(p) + new and s[:len(p)] == p
            logits = dense_logits(example, w, s[:-1])[len(p) - 1:]
            chosen = logits.gather(1, torch.tensor(s[len(p):], device="cuda")[:, None])[:, 0]
            top = logits.amax(1)
            assert (top - chosen <= 64 * ref.ROUNDOFF[dtype] * logits.abs().amax(1)).all()
            same += int((chosen == top).sum())
            total += new
        assert same >= 0.9 * total
