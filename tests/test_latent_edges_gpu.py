"""Latent attention and rotary positions where the other files do not reach: the ends of a CTA's work,
inconsistent start locations, batches and tables of the sizes that take other paths."""

import math
import threading

import pytest
import torch

from _util import bits_equal, cuda_device, seeded, stream
from test_latent_gpu import L, R, SCALE, W, check_attention, check_expanded, paged, reference, reference_expanded
from test_rotary_layout_gpu import U, close, table, turned
from vllm_nt._ntops import capi
from vllm_nt._ntops.torch import (
    latent_attention,
    latent_attention_prefill,
    latent_rope_and_cache,
    rope_cos_sin_cache,
    rotary_embedding,
)
from vllm_nt._ntops.torch._ext import ops

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,rot,first", [
    (20011, 64, 7), (131075, 64, (1 << 20) + 3), (30011, 80, 0),  # 5 (an odd number), 28 and 9 rows a thread
    (1301, 1026, 5),                                              # 3, a frequency a thread
    (500001, 2, 1 << 22), (3000, 128, (1 << 31) - 1000),
])
def test_tables_of_more_rows_than_one_wave_takes_in_pairs(rows, rot, first, dtype):
    got = rope_cos_sin_cache(rows, rot, 500000.0, magnitude=1.25, first_position=first, dtype=dtype, device=cuda_device())
    ref, tol = table_reference(rows, rot, 500000.0, first, 1.25)
    close(got, ref, tol(U[dtype]))


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


# ---- rotations of calls that fill the GPU: four vectors a lane ----


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype,table_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                               (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("tokens,hq,hk,head,rot", [
    (1300, 20, 8, 64, 64), (1200, 33, 1, 128, 128),  # as many vectors a head as divide 32
    (1300, 22, 1, 96, 96), (1250, 3, 8, 80, 48),     # and not
    (1250, 2, 1, 64, 10), (1190, 9, 8, 24, 6),       # pair by pair
])
def test_rotation_of_many_tokens(tokens, hq, hk, head, rot, dtype, table_dtype, interleaved):
    dev = cuda_device()
    g = seeded(tokens + rot)
    q = torch.randn(tokens, hq, head, generator=g).to(dtype)
    k = torch.randn(tokens, hk, head, generator=g).to(dtype)
    pos = torch.randint(0, 5000, (tokens,), generator=g)
    cs = table(5000, rot, table_dtype)
    qd, kd = q.to(dev), k.to(dev)
    ops().rotary_embedding(pos.to(dev), qd, kd, cs.to(dev), head, rot, interleaved)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == 0
    close(qd, *turned(q, cs, pos, rot, interleaved))
    close(kd, *turned(k, cs, pos, rot, interleaved))
    assert bits_equal(qd[..., rot:].cpu(), q[..., rot:]) and bits_equal(kd[..., rot:].cpu(), k[..., rot:])


@pytest.mark.parametrize("interleaved,skew", [(True, 2), (False, 1)])
def test_rotation_of_many_unaligned_rows(interleaved, skew):
    dev = cuda_device()
    g = seeded(65)
    t, h, d = 1300, 9, 64
    wide = torch.randn(t, h, d + 6, generator=g).bfloat16()
    pos = torch.randint(0, 50, (t,), generator=g)
    cs = table(50, d)
    wd = wide.to(dev)
    rotary_embedding(pos.to(dev), wd[..., skew : skew + d], None, d, cs.to(dev), interleaved=interleaved)
    close(wd[..., skew : skew + d], *turned(wide[..., skew : skew + d], cs, pos, d, interleaved))
    assert bits_equal(wd[..., :skew].cpu(), wide[..., :skew])
    assert bits_equal(wd[..., skew + d :].cpu(), wide[..., skew + d :])


# ---- offsets beyond 32 bits ----


def far_apart(t, dim, stride):
    """t's values with `stride` elements from one index of `dim` to the next, in memory of their own."""
    strides = list(t.contiguous().stride())
    strides[dim] = stride
    buf = torch.empty(1 + sum((n - 1) * s for n, s in zip(t.shape, strides)), dtype=t.dtype, device=t.device)
    return buf.as_strided(t.shape, strides).copy_(t)


def test_rotations_beyond_32_bit_offsets():
    dev = cuda_device()
    g = seeded(66)
    q = torch.randn(3, 2, 64, generator=g).bfloat16().to(dev)
    k = torch.randn(3, 1, 64, generator=g).bfloat16().to(dev)
    pos, cs = torch.tensor([5, 0, 40], device=dev), table(50, 64).to(dev)
    for interleaved in (True, False):
        near, far = (q.clone(), k.clone()), (far_apart(q, 0, 1_200_000_000), far_apart(k, 0, 1_200_000_008))
        for x, y in (near, far):
            rotary_embedding(pos, x, y, 64, cs, interleaved=interleaved)
        assert bits_equal(far[0].cpu(), near[0].cpu()) and bits_equal(far[1].cpu(), near[1].cpu())
        assert not bits_equal(near[0].cpu(), q.cpu())


def test_prompts_beyond_32_bit_offsets():
    """Queries and outputs far apart by token, keys and values by head."""
    dev = cuda_device()
    g = seeded(67)
    t, h = 300, 3
    q = torch.randn(t, h, 192, generator=g).bfloat16().to(dev)
    kv = torch.randn(t, h, 256, generator=g).bfloat16().to(dev)
    kr = torch.randn(t, 64, generator=g).bfloat16().to(dev)
    cu = torch.tensor([0, 130, t], dtype=torch.int32, device=dev)
    near = torch.empty(t, h, 128, dtype=torch.bfloat16, device=dev)
    far = far_apart(torch.zeros_like(near), 0, 8_000_000)
    latent_attention_prefill(near, q, kv[..., :128], kr, kv[..., 128:], cu, cu, 170, SCALE)
    wide = far_apart(kv, 1, 1_200_000_000)
    latent_attention_prefill(far, far_apart(q, 0, 8_000_000), wide[..., :128], kr, wide[..., 128:], cu, cu, 170, SCALE)
    assert bits_equal(far.cpu(), near.cpu()) and bool((near != 0).any())


def test_absorbed_queries_beyond_32_bit_offsets():
    dev = cuda_device()
    g = seeded(68)
    lens, h = [70, 300, 5], 20
    cache, pages, _ = paged(lens, 16, torch.bfloat16, g)
    ql, qr = (torch.randn(3, h, n, generator=g).bfloat16().to(dev) for n in (L, R))
    args = (cache.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), pages.to(dev), SCALE)
    near = torch.empty_like(ql)
    far = far_apart(torch.zeros_like(ql), 1, 120_000_000)
    latent_attention(near, ql, qr, *args)
    latent_attention(far, far_apart(ql, 0, 1_200_000_000), far_apart(qr, 0, 1_200_000_000), *args)
    assert bits_equal(far.cpu(), near.cpu())


# ---- calls from two host threads, and compiled ones ----


def layer_inputs(seed, t=40, h=6):
    dev = cuda_device()
    g = seeded(seed)
    x, q = torch.randn(t, W, generator=g).bfloat16().to(dev), torch.randn(t, h, 192, generator=g).bfloat16().to(dev)
    ql = torch.randn(t, h, L, generator=g).bfloat16().to(dev)
    kv = torch.randn(t, h, 256, generator=g).bfloat16().to(dev)
    pages = torch.randperm(8, generator=g)[: -(-t // 16)].to(torch.int32)
    slots = pages[torch.arange(t) // 16].long() * 16 + torch.arange(t) % 16
    lens, cu = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([t], [0, t]))
    return x, q, ql, kv, torch.arange(t, device=dev), slots.to(dev), lens, cu, pages[None].to(dev)


def layer(cs, x, q, ql, kv, pos, slots, lens, cu, pages):
    """A layer's calls on copies of its inputs: what they write."""
    x, q = x.clone(), q.clone()
    t, h = q.shape[:2]
    cache = torch.zeros(8, 16, W, dtype=x.dtype, device=x.device)
    latent_rope_and_cache(pos, q[..., 128:], x[:, :L], x[:, L:], cs, cache, slots)
    absorbed, lse = torch.empty_like(ql), torch.empty(t, h, device=x.device)
    latent_attention(absorbed, ql, q[..., 128:], cache, lens, pages, SCALE, query_start_loc=cu, lse=lse)
    out = torch.empty(t, h, 128, dtype=x.dtype, device=x.device)
    latent_attention_prefill(out, q, kv[..., :128], x[:, L:], kv[..., 128:], cu, cu, 40, SCALE)
    rotary_embedding(pos, ql[..., :64].clone(), None, 64, cs, interleaved=True)
    return x, q, cache, absorbed, lse, out


def test_two_host_threads():
    """Each on a stream of its own: the bits of calls alone."""
    dev = cuda_device()
    cs = rope_cos_sin_cache(64, R, device=dev)
    inputs = [layer_inputs(s) for s in (71, 72)]
    want = [[t.cpu() for t in layer(cs, *i)] for i in inputs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream(dev)):
                for _ in range(50):
                    result = layer(cs, *inputs[n])
                got[n] = [t.cpu() for t in result]
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(bits_equal(x, y) for x, y in zip(a, b))


def test_a_compiled_layer():
    """Traced whole (no graph break) with the registered shapes: the bits of the calls themselves."""
    cs = rope_cos_sin_cache(64, R, device=cuda_device())
    inputs = layer_inputs(73)
    want = layer(cs, *inputs)
    got = torch.compile(layer, backend="aot_eager", fullgraph=True)(cs, *inputs)
    torch.cuda.synchronize()
    assert all(bits_equal(a.cpu(), b.cpu()) for a, b in zip(got, want))


# ---- what the arguments allow and the other tests do not call ----


@pytest.mark.parametrize("heads", [130, 200, 600])  # 3, 4 and 10 groups of heads (more than there are teams)
def test_more_heads_than_two_groups(heads):
    check_attention([300, 0, 17, 70], [1, 2, 0, 1], heads, 32, torch.bfloat16, heads)


def test_many_short_sequences_of_two_groups():
    g = seeded(81)
    lens = torch.randint(0, 60, (300,), generator=g).tolist()
    check_attention(lens, [1] * 300, 100, 16, torch.bfloat16, 82)


@pytest.mark.parametrize("page", [1024, 4096])
def test_pages_longer_than_their_sequences(page):
    check_attention([257, 1, 900], [1, 3, 1], 16, page, torch.float16, page)


def test_one_long_chunk():
    check_attention([700], [600], 20, 64, torch.bfloat16, 83)


def test_expanded_with_many_heads():
    check_expanded([40, 1, 130], [40, 300, 130], 300, torch.bfloat16, 84)


@pytest.mark.parametrize("heads,lens,q_lens", [(16, [3000, 5], [1, 1]), (128, [900, 700, 1], [1, 1, 1]), (8, [500, 90], [70, 3])])
def test_bounds_that_only_size_the_launch(heads, lens, q_lens):
    """Contexts longer than announced, as a captured call meets them when it is replayed later."""
    dev = cuda_device()
    g = seeded(heads)
    cache, pages, rows = paged(lens, 16, torch.bfloat16, g)
    starts = [0] + torch.tensor(q_lens).cumsum(0).tolist()
    ql, qr = (torch.randn(starts[-1], heads, n, generator=g).bfloat16() for n in (L, R))
    ref, ref_lse, tol, lse_tol = reference(ql, qr, rows, starts, SCALE)
    for bound in (1, 64, max(lens), 10**9):
        out, lse = torch.empty_like(ql, device=dev), torch.empty(starts[-1], heads, device=dev)
        latent_attention(out, ql.to(dev), qr.to(dev), cache.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                         pages.to(dev), SCALE, query_start_loc=torch.tensor(starts, dtype=torch.int32, device=dev),
                         max_query_len=max(q_lens), max_seq_len=bound, lse=lse)
        close(out, ref, tol)
        close(lse, ref_lse, lse_tol)
    assert capi.read_device_error(stream()) == 0


def test_expanded_bound_that_only_sizes_the_launch():
    dev = cuda_device()
    g = seeded(85)
    lens = [300, 0, 700, 5]
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    t = sum(lens)
    q, kv = torch.randn(t, 2, 192, generator=g).half().to(dev), torch.randn(t, 2, 256, generator=g).half().to(dev)
    kr = torch.randn(t, 64, generator=g).half().to(dev)
    outs = [torch.empty(t, 2, 128, dtype=torch.float16, device=dev) for _ in range(3)]
    for out, bound in zip(outs, (1, 700, 10**6)):
        latent_attention_prefill(out, q, kv[..., :128], kr, kv[..., 128:], cu, cu, bound, SCALE)
    assert bits_equal(outs[0], outs[1]) and bits_equal(outs[2], outs[1])


def test_queries_shared_by_the_heads():
    """A query broadcast to the heads (a stride of 0) is read as it is."""
    dev = cuda_device()
    g = seeded(86)
    lens, h = [90, 33], 5
    cache, pages, rows = paged(lens, 16, torch.bfloat16, g)
    ql, qr = (torch.randn(2, 1, n, generator=g).bfloat16() for n in (L, R))
    out = torch.empty(2, h, L, dtype=torch.bfloat16, device=dev)
    latent_attention(out, ql.to(dev).expand(2, h, L), qr.to(dev).expand(2, h, R), cache.to(dev),
                     torch.tensor(lens, dtype=torch.int32, device=dev), pages.to(dev), SCALE)
    ref, _, tol, _ = reference(ql.expand(2, h, L), qr.expand(2, h, R), rows, [0, 1, 2], SCALE)
    close(out, ref, tol)
