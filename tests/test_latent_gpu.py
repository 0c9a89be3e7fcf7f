"""GPU parity of the latent-attention operators (ntb200_latent_rope_and_cache,
ntb200_latent_attention) against their definitions in 64 bits.

Tolerances are bounds by arithmetic, element by element.  u is half a step of the storage type
(2^-8 for bf16, 2^-11 for fp16).  An attention output is sum_j w_j c_j with w the softmax of s:
each weight is rounded once to the type and the output once, u * (sum_j w_j |c_j| + |out|); a
score is an fp32 sum of 576 products, off by at most 576 * 2^-24 * scale * sum_d |q_d c_d|, which
moves every weight by twice that relatively; fp16 weights below 2^-14 have an absolute step of
2^-24 while the row's sum is at least 2^7 (the largest weight)."""

import pytest
import torch

from _util import cuda_device, seeded, stream
from vllm_nt._ntops import capi
from vllm_nt._ntops.torch import latent_attention, latent_attention_prefill

pytestmark = pytest.mark.gpu

L, R = 512, 64
W = L + R
SCALE = 192 ** -0.5
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


@pytest.fixture(autouse=True)
def _clean_device_error():
    dev = cuda_device()
    torch.cuda.synchronize(dev)
    capi.read_device_error(stream())
    yield
    torch.cuda.synchronize(dev)


def paged(lens, page, dtype, g, fill=float("nan"), extra=2, pad=0):
    """A cache whose pages hold the sequences' rows in shuffled order and `fill` everywhere else,
    its block table, and the rows themselves.  pad: elements between a token's row and the next."""
    pages = [-(-n // page) for n in lens]
    blocks = sum(pages) + extra
    order = torch.randperm(blocks, generator=g).to(torch.int32)
    cache = torch.full((blocks, page, W + pad), fill, dtype=dtype)
    table = torch.full((len(lens), max(max(pages), 1) + 1), -7, dtype=torch.int32)  # entries past the length are junk
    rows, at = [], 0
    for b, n in enumerate(lens):
        table[b, : pages[b]] = order[at : at + pages[b]]
        at += pages[b]
        x = torch.randn(n, W, generator=g).to(dtype)
        for i in range(pages[b]):
            part = x[i * page : (i + 1) * page]
            cache[table[b, i], : part.shape[0], :W] = part
        rows.append(x)
    return cache, table, rows


def reference(ql, qr, rows, starts, scale):
    """out, lse and the elementwise tolerance, in 64 bits."""
    u = U[ql.dtype]
    q = torch.cat((ql, qr), -1).double()
    t, h, _ = q.shape
    out, lse, tol = torch.zeros(t, h, L).double(), torch.zeros(t, h).double(), torch.zeros(t, h, L).double()
    lse_tol = torch.zeros(t, h).double()
    for b, c in enumerate(rows):
        c = c.double()
        n, q0, q1 = c.shape[0], starts[b], starts[b + 1]
        for i in range(q0, q1):
            seen = c[: max(n - (q1 - q0) + (i - q0) + 1, 0)]
            if seen.shape[0] == 0:
                lse[i] = -torch.inf
                continue
            s = (q[i] @ seen.T) * scale
            ds = W * 2.0**-24 * scale * (q[i].abs() @ seen.abs().T).amax(-1)
            lse[i] = torch.logsumexp(s, -1)
            w = torch.softmax(s, -1)
            mag = w @ seen[:, :L].abs()
            out[i] = w @ seen[:, :L]
            tol[i] = u * (mag + out[i].abs()) + (2 * ds[:, None] + 2.0**-20) * mag
            if ql.dtype == torch.float16:
                tol[i] += seen.shape[0] * 2.0**-32 * seen.abs().max() + 2.0**-25
            lse_tol[i] = ds + (seen.shape[0] + 64) * 2.0**-24 + 2.0**-21 * lse[i].abs()
    return out, lse, tol, lse_tol


def check_attention(lens, q_lens, heads, page, dtype, seed, *, uniform=False, pad=0, tail=3, strided=False,
                    use_lse=True, q_scale=1.0):
    dev = cuda_device()
    g = seeded(seed)
    cache, table, rows = paged(lens, page, dtype, g, pad=pad)
    starts = [0]
    for n in q_lens:
        starts.append(starts[-1] + n)
    t = starts[-1] + (0 if uniform else tail)
    if strided:  # the rotary part inside a wider head, the latent part in its own padded rows
        wide = (torch.randn(t, heads, 192, generator=g) * q_scale).to(dtype)
        big = (torch.randn(t, heads, L + 8, generator=g) * q_scale).to(dtype)
        wide_d, big_d = wide.to(dev), big.to(dev)
        ql, qr, qld, qrd = big[..., :L], wide[..., 128:], big_d[..., :L], wide_d[..., 128:]
        out = torch.full((t, heads, L + 16), 7.0, dtype=dtype, device=dev)[..., :L]
    else:
        ql = (torch.randn(t, heads, L, generator=g) * q_scale).to(dtype)
        qr = (torch.randn(t, heads, R, generator=g) * q_scale).to(dtype)
        qld, qrd = ql.to(dev), qr.to(dev)
        out = torch.full((t, heads, L), 7.0, dtype=dtype, device=dev)
    lse = torch.full((t, heads), 7.0, device=dev) if use_lse else None
    kw = {} if uniform else dict(query_start_loc=torch.tensor(starts, dtype=torch.int32, device=dev),
                                 max_query_len=max(q_lens))
    latent_attention(out, qld, qrd, cache.to(dev)[..., :W], torch.tensor(lens, dtype=torch.int32, device=dev),
                     table.to(dev), SCALE, lse=lse, **kw)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == 0
    n = starts[-1]
    ref, ref_lse, tol, lse_tol = reference(ql[:n], qr[:n], rows, starts, SCALE)
    got = out.cpu().double()
    assert bool((got[n:] == 7.0).all())  # rows behind the last sequence
    err = (got[:n] - ref).abs()
    assert bool((err <= tol).all()), (err - tol).max()
    if use_lse:
        got_lse = lse.cpu().double()
        assert bool((got_lse[n:] == 7.0).all())
        empty = ref_lse == -torch.inf
        assert torch.equal(got_lse[:n] == -torch.inf, empty)
        e = (got_lse[:n] - ref_lse).abs()[~empty]
        assert bool((e <= lse_tol[~empty]).all()), (e - lse_tol[~empty]).max()


EDGES = [1, 0, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [1, 8, 16, 20, 33, 64, 100, 128])
def test_decode_lengths_and_heads(heads, dtype):
    """One query a sequence at every length where a tile, a page or a 16-token step ends, an
    empty context among them; the pages' unused rows hold NaN."""
    check_attention(EDGES, [1] * len(EDGES), heads, 16, dtype, heads)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128])
def test_pages_of_every_size(page):
    check_attention([257, 1, 64, 500], [1, 1, 1, 1], 16, page, torch.bfloat16, page)


@pytest.mark.parametrize("heads,ctx", [(16, 5000), (128, 3000), (40, 9000)])
def test_one_long_context_is_split_and_joined(heads, ctx):
    check_attention([ctx], [1], heads, 64, torch.bfloat16, ctx, uniform=True)


@pytest.mark.parametrize("heads,q_lens", [(16, [2, 1, 5, 3]), (20, [40, 1, 7, 70]), (128, [2, 2, 4, 1]), (1, [130, 64, 1, 65]),
                                          (96, [9, 20, 1, 3])])
def test_chunks_of_new_tokens(heads, q_lens):
    """Several new tokens a sequence, causal: token i sees the cache up to its own position."""
    check_attention([200, 64, 7, 333], q_lens, heads, 32, torch.float16, heads)


def test_more_queries_than_context_leaves_empty_rows():
    check_attention([3, 0, 70], [5, 2, 70], 16, 16, torch.bfloat16, 5)


def test_sequences_without_queries_are_skipped():
    check_attention([30, 50, 0, 70], [1, 0, 0, 3], 16, 16, torch.bfloat16, 6)


def test_uniform_queries_without_start_locations():
    check_attention([100, 31, 64], [3, 3, 3], 32, 16, torch.bfloat16, 7, uniform=True)


def test_strided_queries_outputs_and_cache():
    check_attention([100, 31, 700], [1, 4, 1], 24, 64, torch.float16, 8, strided=True, pad=24)


def test_without_lse():
    check_attention([100, 31], [1, 1], 16, 64, torch.bfloat16, 9, use_lse=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_peaked_scores_rescale_the_output(dtype):
    """Scores over hundreds: the running maximum grows often, and most weights vanish."""
    check_attention([1500, 200], [1, 3], 16, 64, dtype, 10, q_scale=40.0)


@pytest.mark.parametrize("heads", [16, 64])
def test_many_short_sequences_share_a_cta(heads):
    g = seeded(3)
    lens = torch.randint(1, 200, (700,), generator=g).tolist()
    check_attention(lens, [1] * 700, heads, 16, torch.bfloat16, 11)


# ---- the expanded form ----


def reference_expanded(q, kn, kr, v, qs, ks, causal):
    """out, lse and their tolerances in 64 bits (the bounds of `reference`, 192 products a score)."""
    u = U[q.dtype]
    t, h, _ = q.shape
    out, lse, tol = torch.zeros(t, h, 128).double(), torch.zeros(t, h).double(), torch.zeros(t, h, 128).double()
    lse_tol = torch.zeros(t, h).double()
    for b in range(len(qs) - 1):
        q0, q1, k0, k1 = qs[b], qs[b + 1], ks[b], ks[b + 1]
        nq, nk = q1 - q0, k1 - k0
        for j in range(h):
            qq = q[q0:q1, j].double()
            kk = torch.cat((kn[k0:k1, j], kr[k0:k1]), -1).double()
            vv = v[k0:k1, j].double()
            s = qq @ kk.T * SCALE
            hidden = torch.ones(nq, nk, dtype=torch.bool).triu(nk - nq + 1) if causal else torch.zeros(nq, nk, dtype=torch.bool)
            s = s.masked_fill(hidden, -torch.inf)
            ds = 192 * 2.0**-24 * SCALE * (qq.abs() @ kk.abs().T).amax(-1) if nk else torch.zeros(nq).double()
            lse[q0:q1, j] = torch.logsumexp(s, -1)
            w = torch.nan_to_num(torch.softmax(s, -1))
            mag = w @ vv.abs()
            out[q0:q1, j] = w @ vv
            tol[q0:q1, j] = u * (mag + out[q0:q1, j].abs()) + (2 * ds[:, None] + 2.0**-20) * mag
            if q.dtype == torch.float16 and nk:
                tol[q0:q1, j] += nk * 2.0**-32 * vv.abs().max() + 2.0**-25
            lse_tol[q0:q1, j] = ds + (nk + 64) * 2.0**-24 + 2.0**-21 * lse[q0:q1, j].abs()
    return out, lse, tol, lse_tol


def check_expanded(q_lens, k_lens, heads, dtype, seed, *, causal=True, tail=3, separate=False, use_lse=True, q_scale=1.0):
    dev = cuda_device()
    g = seeded(seed)
    qs, ks = [0], [0]
    for a, b in zip(q_lens, k_lens):
        qs.append(qs[-1] + a)
        ks.append(ks[-1] + b)
    t, n, k = qs[-1] + tail, qs[-1], ks[-1] + tail
    q = (torch.randn(t, heads, 192, generator=g) * q_scale).to(dtype)
    kv = torch.randn(k, heads, 256, generator=g).to(dtype)
    kr = torch.randn(k, 64, generator=g).to(dtype)
    kv[ks[-1] :], kr[ks[-1] :], q[n:] = float("nan"), float("nan"), float("nan")  # rows behind the last sequence
    kvd, qd, krd = kv.to(dev), q.to(dev), kr.to(dev)
    knd, vd = kvd[..., :128], kvd[..., 128:]
    if separate:
        knd, vd = knd.contiguous(), vd.contiguous()
    out = torch.full((t, heads, 128), 7.0, dtype=dtype, device=dev)
    lse = torch.full((t, heads), 7.0, device=dev) if use_lse else None
    latent_attention_prefill(out, qd, knd, krd, vd, torch.tensor(qs, dtype=torch.int32, device=dev),
                             torch.tensor(ks, dtype=torch.int32, device=dev), max(q_lens), SCALE, causal, lse)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == 0
    ref, ref_lse, tol, lse_tol = reference_expanded(q[:n], kv[..., :128], kr, kv[..., 128:], qs, ks, causal)
    got = out.cpu().double()
    assert bool((got[n:] == 7.0).all())
    err = (got[:n] - ref).abs()
    assert bool((err <= tol).all()), (err - tol).max()
    if use_lse:
        got_lse = lse.cpu().double()
        assert bool((got_lse[n:] == 7.0).all())
        empty = ref_lse == -torch.inf
        assert torch.equal(got_lse[:n] == -torch.inf, empty)
        e = (got_lse[:n] - ref_lse).abs()[~empty]
        assert bool((e <= lse_tol[~empty]).all()), (e - lse_tol[~empty]).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
def test_expanded_at_tile_edges(causal, dtype):
    """Prompts that end at, before and after a 16-step, a 128-row tile and a 256-row item; the next
    sequence's rows follow directly."""
    lens = [1, 15, 16, 17, 127, 128, 129, 255, 256, 257, 400, 0, 2]
    check_expanded(lens, lens, 3, dtype, 21, causal=causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens,k_lens", [([1, 1, 3], [500, 1, 129]), ([130, 20], [700, 300]), ([300, 5, 64], [100, 0, 64])])
def test_expanded_queries_at_the_end_of_longer_or_shorter_contexts(q_lens, k_lens, causal):
    """Cached prefixes, no keys at all, and more queries than keys (causal: rows that see nothing)."""
    check_expanded(q_lens, k_lens, 5, torch.bfloat16, 22, causal=causal)


@pytest.mark.parametrize("heads", [1, 10, 128])
def test_expanded_heads_and_separate_tensors(heads):
    check_expanded([70, 200], [70, 260], heads, torch.float16, heads, separate=True, use_lse=heads != 10)


def test_expanded_long_prompt():
    check_expanded([2100], [2100], 2, torch.bfloat16, 23)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_expanded_peaked_scores(dtype):
    check_expanded([300, 40], [300, 900], 2, dtype, 24, q_scale=40.0)


def test_expanded_many_short_prompts():
    g = seeded(25)
    lens = torch.randint(0, 40, (150,), generator=g).tolist()
    check_expanded(lens, lens, 3, torch.bfloat16, 26)


def test_expanded_items_where_one_row_tile_sees_nothing():
    """Prompts of both, only the first, and (more queries than keys) only the second tile of rows, and
    of none, in turn through every CTA."""
    q_lens = [256, 100, 300, 20, 512, 130] * 20
    k_lens = [100, 100, 700, 20, 200, 0] * 20
    check_expanded(q_lens, k_lens, 4, torch.bfloat16, 27)
