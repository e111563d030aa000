"""The model's rotation through the operator keeps the eager expression's results, and decode with a 4-bit cache:
graph and eager steps give the same tokens, and a step's attention equals its definition over the records."""
import pytest
import torch

import kv4_plain as P
from openattention_b200 import kv4, llama as L
from openattention_b200 import method as Mth

pytestmark = pytest.mark.gpu
D = 128


def _model(seed, T, steps, layers=2):
    cfg = L.LlamaConfig(layers=layers, ffn=1024, vocab=2048, kv4=True)
    model = L.RandomLlama(cfg, 2, T + steps + 16, "cuda", seed=seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 1)
    prompt = torch.randint(0, cfg.vocab, (2, T), generator=g, device="cuda")
    first = model.prefill(prompt)
    model.start_decode(T, first)
    return model


def _run(graph, steps=6, T=300):
    model = _model(3, T, steps)
    if graph:
        model.capture()
    toks = [(model.step_graph() if graph else model.step_eager()).clone() for _ in range(steps)]
    torch.cuda.synchronize()
    assert int(Mth.C.n_dev.item()) == T + steps
    caches = torch.stack(model.cache4)
    assert not caches[:, :, :, T + steps:].any() and caches[:, :, :, :T + steps].any(-1).all()
    return torch.stack(toks), caches


def test_kv4_graph_decode_matches_eager():
    (a, ca), (b, cb) = _run(False), _run(True)
    assert torch.equal(a, b) and torch.equal(ca, cb)


def test_kv4_decode_layer_matches_definition(monkeypatch):
    """One step, layer 0: the rotated query and the attention row against 64 bits over the layer's records."""
    T = 150
    model = _model(5, T, 1, layers=1)
    seen = {}
    real = kv4.decode_attention

    def spy(q, cache, n, **kw):
        out = real(q, cache, n, **kw)
        seen.update(q=q.cpu(), cache=cache.cpu(), n=int(n), out=out.cpu())
        return out

    monkeypatch.setattr(L.kv4, "decode_attention", spy)
    model.step_eager()
    assert seen["n"] == T + 1
    for b in range(2):
        for h in range(0, 32, 5):
            want, slack = P.attend(seen["q"][b, h, 0], seen["cache"][b, h // 4, :T + 1], D ** -0.5)
            P.check(seen["out"][b, h, 0], want, slack)


def test_prefill_keys_are_the_eager_rotations(monkeypatch):
    """The bf16 cache after a prompt holds, bit for bit, x * cos + rotate(x) * sin of the projected keys."""
    cfg = L.LlamaConfig(layers=1, ffn=256, vocab=512)
    T = 1100
    model = L.RandomLlama(cfg, 1, T + 8, "cuda", rho=0.01, seed=7)
    seen = {}
    real = L.rotary.qk_norm_rope

    def spy(q, k, *a, **kw):
        seen.update(q=q.clone(), k=k.clone())
        seen["out"] = real(q, k, *a, **kw)
        return seen["out"]

    monkeypatch.setattr(L.rotary, "qk_norm_rope", spy)
    model.prefill(torch.arange(T, device="cuda")[None] % cfg.vocab)

    def eager(x):
        f = x.float()
        return (f * model.cos[:T] + torch.cat([-f[..., 64:], f[..., :64]], -1) * model.sin[:T]).to(torch.bfloat16)

    assert torch.equal(seen["out"][0], eager(seen["q"]))
    assert torch.equal(model.K[0][0, :, :T], eager(seen["k"])[0])


@pytest.mark.parametrize("four_bits", [False, True])
def test_tokens_past_the_caches_are_refused(four_bits):
    cfg = L.LlamaConfig(layers=1, ffn=256, vocab=512, kv4=four_bits)
    T = 1030
    model = L.RandomLlama(cfg, 1, T + 2, "cuda", rho=0.01, seed=9)
    with pytest.raises(RuntimeError, match="tokens must be"):
        model.prefill(torch.zeros(1, T + 3, dtype=torch.int64, device="cuda"))
    model.start_decode(T, model.prefill(torch.arange(T, device="cuda")[None] % cfg.vocab))
    model.step_eager()
    model.step_eager()
    with pytest.raises(RuntimeError, match="caches are full"):
        model.step_eager()
    torch.cuda.synchronize()
