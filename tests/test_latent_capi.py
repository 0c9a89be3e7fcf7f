"""Host-side argument checks of the latent-attention and rotary-layout C entry points: bad calls
are refused and empty ones accepted before a device is touched.  CPU only (no kernel runs)."""

import pytest
import torch

from vllm_nt._ntops import capi
from vllm_nt._ntops.torch._ext import ops

# (positions, dtype, query, key, table, table dtype, tokens, q/k heads, head size, rotary dim,
#  interleaved, q token/head, k token/head strides, table row stride, table rows, dtype, stream)
ROTARY = [16, 4, 16, 16, 16, 0, 4, 2, 1, 64, 64, 1, 128, 64, 64, 64, 64, 10, 1, None]
# (out, positions, first, rotary dim, base, scaling, factor, original, beta fast/slow, magnitude,
#  divisors, row stride, dtype, stream)
TABLE = [16, 4, 0, 64, 1e4, 3, 4.0, 4096.0, 32.0, 1.0, 1.0, None, 64, 0, None]
# (positions, dtype, query, latent, key, weight, eps, table, table dtype, interleaved, cache,
#  latent out, slots, dtype, tokens, stored, heads, latent/rope dim, q token/head, latent, key,
#  latent out, table row strides, table rows, block size, slots, block/page strides, dtype, stream)
STORE = [16, 4, 16, 16, 16, 16, 1e-6, 16, 0, 1, 16, 16, 16, 4, 4, 4, 2, 512, 64, 128, 64, 576, 576, 512, 64, 10, 16, 32,
         9216, 576, 1, None]
# (out, lse, q latent, q rope, cache, query_start_loc, seq_lens, block tables, seqs, tokens, heads,
#  latent/rope dim, block size, blocks, max blocks, table stride, max query/seq len, scale,
#  q latent, q rope, out token/head, lse token, cache block/page strides, workspace, bytes, dtype, stream)
LATENT = [16, 16, 16, 16, 16, 16, 16, 16, 2, 4, 16, 512, 64, 16, 8, 4, 4, 2, 64, 0.1, 8192, 512, 1024, 64, 8192, 512, 16,
          9216, 576, 256, 1 << 40, 1, None]
# (out, lse, query, k nope, k rope, value, cu q, cu k, seqs, q/k tokens, heads, dims, max query,
#  scale, causal, q, k nope, (rope), value, out, lse strides, dtype, stream)
PREFILL = [16, 16, 16, 16, 16, 16, 16, 16, 2, 8, 8, 4, 128, 64, 128, 4, 0.1, 1, 768, 192, 1024, 256, 64, 1024, 256, 512, 128,
           4, 1, None]

INVALID, DTYPE, MISALIGNED, WORKSPACE, SHAPE = -1, -2, -3, -4, -6


def refused(name, base, change, status):
    args = list(base)
    for i, v in change.items():
        args[i] = v
    assert getattr(capi.lib(), name)(*args) == status, capi.lib().ntb200_last_error()


@pytest.mark.parametrize("change,status", [
    ({18: 3}, DTYPE), ({5: 2}, DTYPE), ({1: 0}, DTYPE),                       # int heads, fp16 table of bf16 heads, float positions
    ({10: 63}, INVALID), ({10: 0}, INVALID), ({10: 66}, INVALID), ({6: -1}, INVALID), ({16: 32}, INVALID), ({9: 0}, INVALID),
    ({0: None}, INVALID), ({2: None}, INVALID), ({4: None}, INVALID),
    ({7: 1 << 40}, SHAPE), ({2: 18}, MISALIGNED), ({12: 129}, MISALIGNED), ({15: 63}, MISALIGNED),  # a split pair
    ({6: 0}, 0), ({3: None, 7: 0}, 0),
])
def test_rotary(change, status):
    refused("ntb200_rotary_embedding", ROTARY, change, status)


@pytest.mark.parametrize("change,status", [
    ({13: 4}, DTYPE), ({3: 63}, INVALID), ({3: 0}, INVALID), ({1: -1}, INVALID), ({2: -1}, INVALID), ({12: 62}, INVALID),
    ({4: 1.0}, INVALID), ({4: float("nan")}, INVALID), ({6: 0.0}, INVALID), ({6: float("inf")}, INVALID), ({5: 4}, INVALID),
    ({5: -1}, INVALID), ({7: 0.0}, INVALID), ({8: 0.5}, INVALID), ({9: 0.0}, INVALID), ({10: float("inf")}, INVALID),
    ({0: None}, INVALID), ({3: 65538, 12: 65538}, SHAPE), ({2: 1 << 41}, SHAPE), ({1: 0}, 0),
])
def test_table(change, status):
    refused("ntb200_rope_cos_sin_cache", TABLE, change, status)


@pytest.mark.parametrize("change,status", [
    ({30: 0}, DTYPE), ({8: 2}, DTYPE), ({1: 1}, DTYPE), ({13: 0}, DTYPE),
    ({14: -1}, INVALID), ({15: 5}, INVALID), ({26: 0}, INVALID), ({29: 568}, INVALID), ({24: 32}, INVALID), ({21: 504}, INVALID),
    ({0: None}, INVALID), ({3: None}, INVALID), ({4: None}, INVALID), ({7: None}, INVALID), ({10: None}, INVALID),
    ({12: None}, INVALID),
    ({17: 516, 29: 584}, SHAPE), ({17: 1032, 21: 1096, 29: 1096}, SHAPE), ({18: 24}, SHAPE), ({18: 272, 22: 576, 24: 272, 29: 784}, SHAPE),
    ({3: 8}, MISALIGNED), ({10: 8}, MISALIGNED), ({20: 68}, MISALIGNED), ({28: 9220}, MISALIGNED), ({24: 66}, MISALIGNED),
    ({14: 0, 15: 0}, 0),
])
def test_store(change, status):
    refused("ntb200_latent_rope_and_cache", STORE, change, status)


@pytest.mark.parametrize("change,status", [
    ({31: 0}, DTYPE), ({11: 256}, SHAPE), ({12: 32}, SHAPE), ({13: 8}, SHAPE), ({13: 0}, SHAPE), ({10: 65536}, SHAPE),
    ({8: -1}, INVALID), ({19: 0.0}, INVALID), ({19: float("nan")}, INVALID), ({10: 0}, INVALID), ({16: 3}, INVALID), ({17: -1}, INVALID), ({5: None, 9: 5}, INVALID),
    ({0: None}, INVALID), ({2: None}, INVALID), ({3: None}, INVALID), ({4: None}, INVALID), ({6: None}, INVALID),
    ({7: None}, INVALID), ({28: 568}, INVALID),
    ({2: 8}, MISALIGNED), ({20: 8193}, MISALIGNED), ({27: 9220}, MISALIGNED), ({0: 8}, MISALIGNED),
    ({29: None}, WORKSPACE), ({29: 128}, WORKSPACE), ({30: 1024}, WORKSPACE),
    ({8: 0}, 0), ({9: 0}, 0), ({17: 0}, 0),
])
def test_latent(change, status):
    refused("ntb200_latent_attention", LATENT, change, status)


@pytest.mark.parametrize("change,status", [
    ({28: 0}, DTYPE), ({12: 64}, SHAPE), ({13: 32}, SHAPE), ({14: 192}, SHAPE), ({11: 65536}, SHAPE),
    ({8: -1}, INVALID), ({9: -1}, INVALID), ({11: 0}, INVALID), ({16: 0.0}, INVALID), ({16: -0.1}, INVALID),
    ({16: float("nan")}, INVALID), ({0: None}, INVALID), ({2: None}, INVALID), ({3: None}, INVALID), ({4: None}, INVALID),
    ({5: None}, INVALID), ({6: None}, INVALID), ({7: None}, INVALID),
    ({2: 8}, MISALIGNED), ({20: 1028}, MISALIGNED), ({22: 68}, MISALIGNED), ({25: 516}, MISALIGNED),
    ({8: 0}, 0), ({9: 0}, 0), ({15: 0}, 0),
])
def test_prefill(change, status):
    refused("ntb200_latent_attention_prefill", PREFILL, change, status)


def test_host_tensors_are_refused():
    bf = torch.bfloat16
    x, pos = torch.zeros(2, 1, 64, dtype=bf), torch.zeros(2, dtype=torch.int64)
    calls = [
        lambda: ops().rotary_embedding(pos, x, None, torch.zeros(4, 64), 64, 64, True),
        lambda: ops().rope_cos_sin_cache(torch.zeros(4, 64), 0, 64, 1e4, 0, 1.0, 0.0, 32.0, 1.0, 1.0, None),
        lambda: ops().latent_rope_and_cache(pos, x, torch.zeros(2, 512, dtype=bf), x[:, 0], None, 1e-6, torch.zeros(4, 64),
                                            True, torch.zeros(1, 16, 576, dtype=bf), None, pos),
        lambda: ops().latent_attention(torch.zeros(2, 1, 512, dtype=bf), None, torch.zeros(2, 1, 512, dtype=bf), x,
                                       torch.zeros(1, 16, 576, dtype=bf), None, torch.ones(2, dtype=torch.int32),
                                       torch.zeros(2, 1, dtype=torch.int32), 1, 0, 0.1, None),
        lambda: ops().latent_attention_prefill(torch.zeros(2, 1, 128, dtype=bf), None, torch.zeros(2, 1, 192, dtype=bf),
                                               torch.zeros(2, 1, 128, dtype=bf), x[:, 0], torch.zeros(2, 1, 128, dtype=bf),
                                               torch.tensor([0, 2], dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32),
                                               2, 0.1, True),
    ]
    for call in calls:
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
