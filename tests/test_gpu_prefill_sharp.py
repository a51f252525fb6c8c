"""GPU prefill where a few keys decide: cached keys so large that scores differ by more
than fp16 exponents reach (e^11), at every key position of a tile.  A running maximum
that misses some of a tile's keys lets their weights overflow; the logits must be
finite and those of the decode steps, whose scores are rounded to fp16 (2^-11 of a
score of up to 64 changes a weight by 3 %, hence the 10 %)."""
import numpy as np
import pytest

import cuqwen_amd as cq
from tests.conftest import tiny_config
from tests.gpu_util import rel_err

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", [cq.KV_FP16, cq.KV_INT8])
@pytest.mark.parametrize("hd,rows", [(64, 0), (64, 64), (64, 128), (64, 256), (128, 0)])
def test_sharp_attention(kv, hd, rows):
    cfg = tiny_config(head_dim=hd, dim=4 * hd)
    w = cq.synth_weights(cfg, 77)
    rng = np.random.default_rng(hd)
    toks = rng.integers(0, cfg.vocab_size, 20).tolist()
    st = [cq.State(cfg, w, kv_dtype=kv) for _ in range(2)]
    for layer in range(cfg.n_layers):
        for h in range(cfg.n_kv_heads):
            k = rng.standard_normal((64, hd)).astype(np.float16)
            k[5:64:7] *= np.float16(40)      # one key in each row of lanes, some of them far above the others
            v = rng.standard_normal((64, hd)).astype(np.float16)
            for s in st:
                s.kv_write(layer, h, 0, k)
                s.kv_write(layer, h, 1, v)
    if rows:
        st[0].set_prefill_form(0, 1, rows, 1)
    st[0].prefill(toks, 64)
    for i, t in enumerate(toks):
        st[1].forward(t, 64 + i)
    a, b = (s.logits().astype(np.float64) for s in st)
    assert np.isfinite(a).all(), "overflow"
    assert rel_err(a, b) <= 0.1
    for s in st:
        s.free()
    w.free()
