"""The speculative decoding example: what it caches and computes against a dense fp64 run of its model."""

import importlib.util
import pathlib

import pytest
import torch

from conftest import has_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    if not has_gpu():
        pytest.skip("no CUDA device")
    path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "speculative_decode.py"
    spec = importlib.util.spec_from_file_location("speculative_decode", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def dense(model, tokens):
    """Logits, keys and values of one sequence, causal, in 64 bits."""
    kv = []

    def attend(layer, q, k, v):
        kv.append((k, v))
        k, v = (x.repeat_interleave(model.q_heads // model.heads, 1) for x in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * model.dim ** -0.5
        s = s.masked_fill(torch.ones_like(s[0], dtype=torch.bool).triu(1), -torch.inf)
        return torch.einsum("hij,jhd->ihd", s.softmax(-1), v)
    pos = torch.arange(len(tokens), device=tokens.device).double()
    return model(tokens, pos, attend), kv


# fp32: sums of up to 2048 products through 3 layers, about 2^-24 sqrt(2048) a layer of
# values near 1, with room for their growth: 1e-4.  int8: half a code of 127 in K and V of each
# layer, averaged in the sums: 0.05.
@pytest.mark.parametrize("cache,tol", [("f32", 1e-4), ("i8", 0.05)])
def test_rounds_match_a_dense_run(example, cache, tol):
    target = example.Decoder(300, 256, 3, 4, 2, seed=3)
    draft = example.Decoder(300, 256, 1, 4, 4, seed=4)
    prompts = [[(5 * i + b) % 300 for i in range(n)] for b, n in enumerate((2, 17, 60))]
    run = example.Generator(target, draft, prompts, cache, drafts=3, rounds=6, seed=5)
    for _ in range(6):
        before = run.n
        out, accepted = run.round()
        assert ((accepted >= 0) & (accepted <= 3)).all() and (run.n == before + accepted + 1).all()
    example.paged.check_stream()
    logits = run.logits.view(3, 4, -1)
    cu = torch.nn.functional.pad(before.cumsum(0), (1, 0)).to(torch.int32)
    got_kv = [run.caches[0].read(i, cu, int(cu[-1])) for i in range(3)]
    for b, p in enumerate(prompts):
        n = int(before[b])
        assert run.tokens[b, :len(p)].tolist() == p
        # logits of the last round up to the accepted drafts, and the cache up to its first token
        keep = int(accepted[b]) + 1
        want, kv = dense(target, run.tokens[b, :n - 1 + keep])
        assert float((logits[b, :keep] - want[n - 1:]).abs().max()) <= tol * float(want.abs().max())
        for layer in range(3):
            for x, y in zip(got_kv[layer], kv[layer]):
                assert float((x[int(cu[b]):int(cu[b + 1])] - y[:n]).abs().max()) <= tol * float(y.abs().max())
