"""The prefill attention on the tensor cores gives the same bits each time: its two warps of a row write their
probabilities over scores that both read twice."""
import numpy as np
import pytest

from pyxis_b200 import synth_tokens
from pyxis_b200.model import Decoder, ModelConfig, SyntheticModel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head_dim", [64, 128])
def test_prefill_repeats_bit_for_bit(head_dim):
    cfg = ModelConfig(hidden=256, n_layers=1, n_q_heads=16, n_kv_heads=8, head_dim=head_dim, ffn=512, vocab=2048, rope_theta=1e6)
    dec = Decoder(SyntheticModel(cfg, seed=47, head_norm_value=2.0), qtype="int8", max_seq=1500)
    prompts = synth_tokens(0x77, 4 * 1490, cfg.vocab).reshape(4, 1490)
    first = dec.prefill_hidden(prompts).copy()
    for _ in range(30):
        assert np.array_equal(dec.prefill_hidden(prompts), first)
    dec.close()
