"""Views of foreign memory as operands of calls that are older than views."""
import numpy as np
import pytest

from yuuka_b200 import cuda, synth

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = cuda.Device(0)
    yield d
    d.close()


def test_draft_probs_between_words_are_refused(dev):
    cfg = synth.tiny_config()
    model = cuda.Model(dev, cfg, synth.make_model(cfg, "q8_0", seed=7, unit_norms=False))
    sess = cuda.Session(model, max_batch=1, max_nodes=4, capacity=64, kv_format=cuda.KV_F16)
    sess.forward(np.arange(5, dtype=np.int32), seq=0)
    store = dev.alloc(4 * 4 * cfg["vocab"] + 16)
    tokens, parent, u = np.zeros((1, 4), np.int32), np.array([-1, 0, 1, 2], np.int32), np.full((1, 4, 2), 0.5, np.float32)
    for off in (1, 2, 3):
        view = dev.view(cuda.lib().yuuka_buffer_ptr(store.h) + off, 4 * 4 * cfg["vocab"])
        with pytest.raises(cuda.YuukaError, match="draft_probs does not start at a multiple of 4"):
            sess.verify(tokens, parent=parent, mode=cuda.ACCEPT_REJECTION, temperature=0.8, draft_probs=view, uniforms=u)
        view.free()
    sess.close()
    model.close()
    store.free()


def test_logits_may_start_at_any_word(dev):
    """Rows 4, 8 and 12 bytes behind a multiple of 16 are read like aligned ones."""
    stream, V, N = dev.stream(), 4096, 5
    x = np.random.default_rng(3).standard_normal((1, N, V)).astype(np.float32)
    tokens = np.argmax(x[0], -1)[None, [0, 0, 1, 2, 3]].astype(np.int32)
    store = dev.alloc(x.nbytes + 16)
    got = []
    for off in (0, 4, 8, 12):
        view = dev.view(cuda.lib().yuuka_buffer_ptr(store.h) + off, x.nbytes)
        view.write(x)
        got.append(cuda.accept_tree(stream, view, tokens, V))
        view.free()
    for other in got[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(got[0], other))
    assert got[0][0][0] == N - 1
    store.free()
    stream.destroy()
