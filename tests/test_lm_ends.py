"""The benchmark language model with the operators at its ends injected: on CPU with plain functions
in their place, on a GPU with the library's, alone, captured and as one training step."""
import sys
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))

from baseline import lm  # noqa: E402
from oracle import attnres_oracle as ao  # noqa: E402


def _plain_ends():
    return lm.Ends(
        embed=lambda tokens, table, positions, dtype: (F.embedding(tokens, table) + positions).to(dtype),
        layer_norm=lambda x, w, b, eps: F.layer_norm(x, (x.shape[-1],), w, b, eps),
        loss=lambda h, w, t: F.cross_entropy((h @ w.t()).flatten(0, 1), t.flatten()))


def _models(mode, ends, operator, device="cpu", normed=None, **sizes):
    torch.manual_seed(6)
    config = lm.LMConfig(**{**dict(layers=2, width=16, heads=4, ffn=32, vocab=31, sequence=8, mode=mode,
                                   block_layers=1), **sizes})
    with torch.device(device):
        plain = lm.CausalLM(config, operator, normed_operator=normed)
        twin = lm.CausalLM(config, operator, normed_operator=normed, ends=ends)
    twin.load_state_dict(plain.state_dict())
    tokens = torch.randint(config.vocab, (4, config.sequence), device=device)
    targets = torch.randint(config.vocab, (4, config.sequence), device=device)
    return plain, twin, tokens, targets


@pytest.mark.parametrize("mode", ["full", "block"])
def test_injected_ends_change_nothing(mode):
    plain, twin, tokens, targets = _models(mode, _plain_ends(), lambda v, q: ao.oracle(v, q))
    torch.testing.assert_close(twin(tokens), plain(tokens))
    expected = F.cross_entropy(plain(tokens).flatten(0, 1), targets.flatten())
    torch.testing.assert_close(twin(tokens, targets), expected)
    steps = []
    for model, inside in ((plain, False), (twin, True)):
        optimizer = torch.optim.SGD(model.parameters(), lr=0.1)
        loss = lm.training_step(model, optimizer, tokens, targets, accumulation=2, loss_in_model=inside)
        steps.append((loss, model.state_dict()))
    torch.testing.assert_close(steps[0][0], steps[1][0])
    for name, value in steps[0][1].items():
        torch.testing.assert_close(steps[1][1][name], value, msg=name)


@pytest.mark.gpu
@pytest.mark.parametrize("fused_norm", [False, True], ids=["separate norm", "fused norm"])
def test_library_ends_in_a_training_step(fused_norm):
    """Loss and every parameter's gradient of one BF16-autocast step against the framework's own
    embedding, LayerNorm and head.  The two round BF16 tensors at other places (the framework keeps
    the logits in BF16: 2^-9 of each), so a gradient agrees to a few BF16 steps of its norm."""
    from attnres import _native, attnres
    from attnres.fused import attnres_layer_norm
    plain, twin, tokens, targets = _models(
        "full", lm.library_ends(), attnres, "cuda", attnres_layer_norm if fused_norm else None,
        width=512, heads=8, ffn=1024, vocab=3001, sequence=128)
    losses = []
    for model, inside in ((plain, False), (twin, True)):
        for p in model.parameters():
            p.grad = torch.zeros_like(p)
        optimizer = torch.optim.SGD(model.parameters(), lr=0.0)
        losses.append(lm.training_step(model, optimizer, tokens, targets, loss_in_model=inside))
    torch.testing.assert_close(losses[1], losses[0], rtol=2**-10, atol=0)
    for (name, a), b in zip(plain.named_parameters(), twin.parameters()):
        off = (a.grad.double() - b.grad.double()).norm() / a.grad.double().norm()
        assert off < 2**-5, (name, off.item())
    torch.cuda.synchronize()
    assert _native.error_flag() == 0


@pytest.mark.gpu
def test_library_ends_in_a_captured_step():
    """The whole step in one CUDA graph, replayed: the parameters move as eager steps move them."""
    from attnres import attnres
    eager, captured, tokens, targets = _models("block", lm.library_ends(), attnres, "cuda", width=256,
                                               heads=4, ffn=512, vocab=1003, sequence=64)
    eager.ends = captured.ends
    optimizers = [lm.make_optimizer(m, capturable=True, lr=1e-3) for m in (eager, captured)]
    graph = lm.CapturedStep(
        lambda: lm.training_step(captured, optimizers[1], tokens, targets, loss_in_model=True),
        captured, optimizers[1])
    for _ in range(3):
        lm.training_step(eager, optimizers[0], tokens, targets, loss_in_model=True)
        graph.replay()
    torch.cuda.synchronize()
    for (name, a), b in zip(eager.named_parameters(), captured.named_parameters()):
        torch.testing.assert_close(a, b[1], rtol=0, atol=0, msg=name)


@pytest.mark.gpu
def test_library_ends_compile():
    from attnres import attnres
    _, model, tokens, targets = _models("block", lm.library_ends(), attnres, "cuda", width=256, heads=4,
                                        ffn=512, vocab=1003, sequence=64)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        expected = model(tokens, targets)
        expected.backward()
        wanted = [p.grad.clone() for p in model.parameters()]
        for p in model.parameters():
            p.grad = None
        loss = torch.compile(model, fullgraph=True, dynamic=False)(tokens, targets)
    loss.backward()
    torch.testing.assert_close(loss, expected, rtol=2**-9, atol=0)
    for p, want in zip(model.parameters(), wanted):
        off = (p.grad.double() - want.double()).norm() / want.double().norm()
        assert off < 2**-5, off.item()


@pytest.mark.gpu
def test_network_ends_example_runs():
    import importlib.util
    path = ROOT / "fast-attnres_b200" / "examples" / "network_ends.py"
    spec = importlib.util.spec_from_file_location("example_network_ends", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert module.run("cuda")["gradients"] == 7
