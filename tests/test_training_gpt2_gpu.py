"""GPT-2's token table under training: what reads it after a step in place."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,kmajor,rows", [("float32", False, (3, 30)), ("float32", False, (1, 9)),
                                               ("float16", True, (1, 9)), ("float16", True, (3, 30)),
                                               ("bfloat16", False, (3, 30))])
def test_a_step_on_the_table_is_seen_by_the_head(gpu, dtype, kmajor, rows):
    """The score's logits, by packed copies of the table or by itself, are those
    of the loss again once the copies are made anew; captured heads follow."""
    from applegpu_runtime.models import gpt2 as G
    cfg = dict(n_layer=1, n_head=2, n_embd=128, vocab_size=211, n_positions=96)
    model = G.load_model(G.random_weights(cfg, seed=5, std=0.15), cfg, dtype, kmajor=kmajor)
    ids = np.random.default_rng(0).integers(0, 211, rows).astype(np.int32)
    wte = model["weights"]["transformer.wte.weight"]
    loss, _, dw = G.gpt2_loss(model, ids, grads=True)
    first = loss.to_numpy()
    idx = gpu.from_numpy(ids[0])
    pos = gpu.from_numpy(np.arange(len(ids[0]), dtype=np.int32))
    graph = gpu.capture(lambda: G.gpt2_forward(model, idx, positions=pos)[0])
    gpu.muon_step_(wte, gpu.zeros([211, 128]), dw, lr=0.5)
    G.repack_table(model)
    loss = G.gpt2_loss(model, ids).to_numpy()
    lp = G.gpt2_score(model, ids)[0].to_numpy()
    assert np.abs(loss - first).max() > 0.1
    # logits are rounded to the model's type, float32's products to 2^-16 of
    # their terms
    bar = {"float32": 2.0 ** -13, "float16": 2.0 ** -9, "bfloat16": 2.0 ** -6}[dtype]
    np.testing.assert_allclose(loss, -lp, atol=bar * 16, rtol=bar)
    graph.replay()
    np.testing.assert_array_equal(graph.outputs.to_numpy(), G.gpt2_forward(model, ids[0])[0].to_numpy())
    graph.destroy()
