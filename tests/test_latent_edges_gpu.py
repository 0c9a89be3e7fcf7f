"""Latent attention and rotary positions where the other files do not reach: the ends of a CTA's work,
inconsistent start locations, batches and tables of the sizes that take other paths."""

import pytest
import torch

from _util import bits_equal, cuda_device, seeded, stream
from test_latent_gpu import SCALE, check_expanded
from vllm_nt._ntops import capi
from vllm_nt._ntops.torch import latent_attention_prefill

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_device_error():
    dev = cuda_device()
    torch.cuda.synchronize(dev)
    capi.read_device_error(stream())
    yield
    torch.cuda.synchronize(dev)


# ---- prompts: the last key tile of a CTA, visited by one tile of rows only ----


@pytest.mark.parametrize("q_lens,k_lens,causal", [
    ([100], [385], False), ([128] * 3, [384, 700, 1100], False),     # at most 128 rows: tile A alone
    ([500], [500], True), ([256, 130], [900, 1100], True),          # the second rows see one key tile more
    ([300], [170], True),                                           # only the second rows see keys at all
])
def test_expanded_last_keys_for_one_tile_of_rows(q_lens, k_lens, causal):
    check_expanded(q_lens, k_lens, 3, torch.bfloat16, 61, causal=causal)


def test_expanded_last_keys_for_one_tile_of_rows_repeat_their_bits():
    """Items of 100 rows and three to nine key tiles, one or several a CTA, called again and again."""
    dev = cuda_device()
    g = seeded(62)
    for seqs in (9, 60):
        k_lens = [300 + 90 * (b % 10) for b in range(seqs)]
        q = torch.randn(100 * seqs, 8, 192, generator=g).bfloat16().to(dev)
        kv = torch.randn(sum(k_lens), 8, 256, generator=g).bfloat16().to(dev)
        kr = torch.randn(sum(k_lens), 64, generator=g).bfloat16().to(dev)
        cu_q = torch.arange(0, 100 * seqs + 1, 100, dtype=torch.int32, device=dev)
        cu_k = torch.tensor([0] + torch.tensor(k_lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)
        outs = []
        for _ in range(40):
            out = torch.full((100 * seqs, 8, 128), 7.0, dtype=torch.bfloat16, device=dev)
            latent_attention_prefill(out, q, kv[..., :128], kr, kv[..., 128:], cu_q, cu_k, 100, SCALE)
            outs.append(out)
        torch.cuda.synchronize()
        assert capi.read_device_error(stream()) == 0
        for out in outs[1:]:
            assert bits_equal(out, outs[0])
