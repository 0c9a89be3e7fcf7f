"""Latent attention and rotary positions where the other files do not reach: the ends of a CTA's work,
inconsistent start locations, batches and tables of the sizes that take other paths."""

import math

import pytest
import torch

from _util import bits_equal, cuda_device, seeded, stream
from test_latent_gpu import L, R, SCALE, check_expanded, paged, reference, reference_expanded
from test_rotary_layout_gpu import U, close
from vllm_nt._ntops import capi
from vllm_nt._ntops.torch import (
    latent_attention,
    latent_attention_prefill,
    rope_cos_sin_cache,
)

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


# ---- start locations that fall ----

FAR = 2_000_000_000


@pytest.mark.parametrize("heads", [1, 16, 100])
@pytest.mark.parametrize("starts,right", [
    ([0, 5, 3, 8], 1), ([0, 8, 3, 5], 1), ([0, 2, 5, 0, 8], 2), ([3, 1, 4, 8], 0),
    (list(range(9)) + [2] + list(range(3, 9)), 8), ([0, 5, FAR, -FAR, 3, 8], 1),
    ([0] * 300 + [4, 6, 5, 8] + [8] * 300, 301),  # past the first sequence of every thread
], ids=["5-3", "8-3", "5-0", "at once", "all again", "far", "303rd"])
def test_sequences_behind_a_falling_start_location_are_skipped(starts, right, heads):
    """The first `right` sequences are right, and the rows that they do not own stay as they were: those
    behind the fall could own rows of theirs."""
    dev = cuda_device()
    g = seeded(63)
    n = len(starts) - 1
    lens = [int(x) for x in torch.randint(0, 400 if n < 20 else 40, (n,), generator=g)]
    cache, table, rows = paged(lens, 16, torch.bfloat16, g)
    ql = torch.randn(8, heads, L, generator=g).bfloat16()
    qr = torch.randn(8, heads, R, generator=g).bfloat16()
    out = torch.full((8, heads, L), 7.0, dtype=torch.bfloat16, device=dev)
    lse = torch.full((8, heads), 7.0, device=dev)
    latent_attention(out, ql.to(dev), qr.to(dev), cache.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                     table.to(dev), SCALE, query_start_loc=torch.tensor(starts, dtype=torch.int32, device=dev), lse=lse)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == capi.DEVERR_INDEX_RANGE
    own = starts[right] if right else 0
    assert bool((out[own:] == 7.0).all()) and bool((lse[own:] == 7.0).all())
    if own:
        ref, ref_lse, tol, lse_tol = reference(ql[:own], qr[:own], rows[:right], starts[: right + 1], SCALE)
        close(out[:own], ref, tol)
        seen = ref_lse > -torch.inf
        assert torch.equal(lse[:own].cpu() > -torch.inf, seen)
        close(lse[:own].cpu()[seen], ref_lse[seen], lse_tol[seen])


@pytest.mark.parametrize("cu_q,right", [
    ([0, 20, FAR, -FAR, 5, 30], 1), ([0, 20, FAR, -FAR, 0, 20], 1), ([0, 7, 20, 19, 40], 2),
    ([0] * 40 + [20, FAR, -FAR] + [5, 30] * 20, 40),  # (in a later 32)
], ids=["far", "far, the same", "by one", "42nd"])
def test_prompts_behind_a_fall_between_far_locations_are_skipped(cu_q, right):
    """The difference of the far locations is positive in 32 bits."""
    dev = cuda_device()
    g = seeded(64)
    n, own = len(cu_q) - 1, cu_q[right]
    cu_k = list(cu_q[: right + 1]) + [own] * (n - right)
    q = torch.randn(40, 2, 192, generator=g).half()
    kv = torch.randn(40, 2, 256, generator=g).half()
    kr = torch.randn(40, 64, generator=g).half()
    kvd = kv.to(dev)
    out = torch.full((40, 2, 128), 7.0, dtype=torch.float16, device=dev)
    latent_attention_prefill(out, q.to(dev), kvd[..., :128], kr.to(dev), kvd[..., 128:],
                             torch.tensor(cu_q, dtype=torch.int32, device=dev),
                             torch.tensor(cu_k, dtype=torch.int32, device=dev), 30, SCALE)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == capi.DEVERR_INDEX_RANGE
    ref, _, tol, _ = reference_expanded(q[:own], kv[..., :128], kr, kv[..., 128:], cu_q[: right + 1], cu_k[: right + 1], True)
    close(out[:own], ref, tol)
    assert bool((out[own:] == 7.0).all())


# ---- the table ----


def table_reference(rows, rot, base, first, mag, div=None):
    """The unscaled table in 64 bits, and its tolerance.

    A frequency comes from ln(base) by a handful of fp64 steps whose errors the exponent
    multiplies by ln(base): under 7 ln(base) + 13 halves of a last place, and this one's under
    ln(base) + 4.  The rest beside a quarter turn goes to fp32 with three roundings of at most
    pi / 4, under 2^-23; the series' steps are off by under 2^-23 of 1.  Then the magnitude's product and
    the rounding to the type."""
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if div is not None:
        f = f / div.double()
    a = (first + torch.arange(rows, dtype=torch.float64))[:, None] * f
    ref = mag * torch.cat((a.cos(), a.sin()), -1)
    angle = torch.cat((a, a), -1).abs()
    return ref, lambda u: (mag * (2.0**-22 + (8 * math.log(base) + 17) * 2.0**-53 * angle)
                           + (u + 2.0**-24) * ref.abs() + 2.0**-25 * (u == U[torch.float16]))


@pytest.mark.parametrize("rot", [64, 1026])
def test_divisors_without_a_frequency(rot):
    """f / 0 and f / NaN are no frequency: the columns are NaN, as cos and sin of inf and NaN are.
    f / inf is 0 and -f turns the other way."""
    dev = cuda_device()
    div = torch.ones(rot // 2)
    div[[0, 3, 9, 20, 31]] = torch.tensor([0.0, float("inf"), float("nan"), -2.0, -0.0])
    got = rope_cos_sin_cache(100, rot, freq_divisors=div.to(dev), magnitude=1.5, device=dev).cpu()
    ref, tol = table_reference(100, rot, 10000.0, 0, 1.5, div)
    none = torch.zeros(rot, dtype=torch.bool)
    none[[i + h for i in (0, 9, 31) for h in (0, rot // 2)]] = True
    assert bool(ref[:, none].isnan().all()) and bool(got[:, none].isnan().all())
    close(got[:, ~none], ref[:, ~none], tol(U[torch.float32])[:, ~none])
