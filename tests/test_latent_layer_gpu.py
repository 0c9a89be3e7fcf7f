"""The latent-attention operators together, as one layer uses them -- table, store of a prompt,
attention over its expanded keys, store and absorbed attention of later tokens, a chunk over the
cache -- and the ways a serving loop calls them: captured in CUDA graphs, on side streams, with
a workspace of its own, with padded batches and bad page ids.

Every stage is checked against its definition in 64 bits on the stage's own inputs (what the
device holds after the stage before), with the tolerances of test_latent_gpu.py and
test_rotary_layout_gpu.py."""

import pytest
import torch

from _util import bits_equal, cuda_device, seeded, stream
from test_latent_gpu import L, R, SCALE, W, paged, reference, reference_expanded
from test_rotary_layout_gpu import EPS, close, store_reference, turned
from vllm_nt._ntops import capi
from vllm_nt._ntops.torch import (
    latent_attention,
    latent_attention_prefill,
    latent_rope_and_cache,
    latent_workspace_bytes,
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


def test_a_layer_prefills_decodes_and_takes_a_chunk():
    dev = cuda_device()
    g = seeded(31)
    dt, h, page = torch.bfloat16, 5, 16
    lens = [37, 130, 1]
    w_k = (torch.randn(h, 128, L, generator=g) * L**-0.5).to(dt).to(dev)
    w_v = (torch.randn(h, 128, L, generator=g) * L**-0.5).to(dt).to(dev)
    norm_w = (1 + 0.2 * torch.randn(L, generator=g)).to(dt).to(dev)
    cs = rope_cos_sin_cache(4096, R, scaling="yarn", factor=4.0, original_max_position=1024, magnitude=1.0)
    blocks = 32
    cache = torch.full((blocks, page, W), float("nan"), dtype=dt, device=dev)
    order = torch.randperm(blocks, generator=g).tolist()
    table = torch.tensor([order[10 * b : 10 * b + 10] for b in range(3)], dtype=torch.int32)
    rows = [torch.empty(0, W, dtype=dt) for _ in lens]  # what each sequence has cached

    def step(counts):
        """New tokens for every sequence: their projections, then the store; returns the queries."""
        t = sum(counts)
        x = torch.randn(t, W, generator=g).to(dt)
        q = torch.randn(t, h, 192, generator=g).to(dt)
        pos = torch.cat([torch.arange(rows[b].shape[0], rows[b].shape[0] + n) for b, n in enumerate(counts)])
        which = torch.cat([torch.full((n,), b) for b, n in enumerate(counts)])
        slots = table[which, pos // page].long() * page + pos % page
        xd, qd, normed = x.to(dev), q.to(dev), torch.empty(t, L, dtype=dt, device=dev)
        latent_rope_and_cache(pos.to(dev), qd[..., 128:], xd[:, :L], xd[:, L:], cs, cache, slots.to(dev),
                              norm_weight=norm_w, eps=EPS, latent_out=normed)
        table_host = cs.cpu()
        close(normed, *store_reference(x[:, :L], norm_w.cpu()))
        close(xd[:, None, L:], *turned(x[:, None, L:], table_host, pos, R, True))
        close(qd[..., 128:], *turned(q[..., 128:], table_host, pos, R, True))
        new = torch.cat((normed, xd[:, L:]), -1).cpu()
        assert bits_equal(cache.view(-1, W)[slots.to(dev)].cpu(), new)
        for b in range(3):
            rows[b] = torch.cat((rows[b], new[which == b]))
        return qd, normed, xd[:, L:]

    def absorbed(qd, counts):
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        ql = torch.einsum("thd,hdl->thl", qd[..., :128].float(), w_k.float()).to(dt)
        out, lse = torch.empty_like(ql), torch.empty(ql.shape[:2], device=dev)
        latent_attention(out, ql, qd[..., 128:], cache, torch.tensor([r.shape[0] for r in rows], dtype=torch.int32, device=dev),
                         table.to(dev), SCALE, query_start_loc=torch.tensor(starts, dtype=torch.int32, device=dev),
                         max_query_len=max(counts), lse=lse)
        ref, ref_lse, tol, lse_tol = reference(ql.cpu(), qd[..., 128:].cpu(), rows, starts, SCALE)
        close(out, ref, tol)
        close(lse, ref_lse, lse_tol)
        return out

    # the prompts: keys and values expanded from the normalised latents
    qd, normed, key = step(lens)
    k_nope = torch.einsum("tl,hdl->thd", normed.float(), w_k.float()).to(dt)
    value = torch.einsum("tl,hdl->thd", normed.float(), w_v.float()).to(dt)
    cu = torch.tensor([0, 37, 167, 168], dtype=torch.int32, device=dev)
    out, lse = torch.empty(168, h, 128, dtype=dt, device=dev), torch.empty(168, h, device=dev)
    latent_attention_prefill(out, qd, k_nope, key, value, cu, cu, 130, SCALE, lse=lse)
    ref, ref_lse, tol, lse_tol = reference_expanded(qd.cpu(), k_nope.cpu(), key.cpu(), value.cpu(), cu.tolist(), cu.tolist(), True)
    close(out, ref, tol)
    close(lse, ref_lse, lse_tol)
    # two decode steps, then a chunk for two of the sequences
    for counts in ([1, 1, 1], [1, 1, 1], [7, 0, 20]):
        qd, _, _ = step(counts)
        absorbed(qd, counts)
    assert capi.read_device_error(stream()) == 0


def _decode_case(seed, lens, heads, page=32, dtype=torch.bfloat16):
    dev = cuda_device()
    g = seeded(seed)
    cache, table, rows = paged(lens, page, dtype, g)
    ql = torch.randn(len(lens), heads, L, generator=g).to(dtype)
    qr = torch.randn(len(lens), heads, R, generator=g).to(dtype)
    args = dict(q_latent=ql.to(dev), q_rope=qr.to(dev), kv_cache=cache.to(dev),
                seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev), block_table=table.to(dev), scale=SCALE)
    return args, torch.empty(len(lens), heads, L, dtype=dtype, device=dev)


def test_captured_decodes_with_their_own_and_a_shared_workspace():
    """Two captured calls, replayed after their inputs changed in place; then both once more with one
    workspace between them, in stream order."""
    dev = cuda_device()
    cases = [_decode_case(41, [900, 3, 200], 16), _decode_case(42, [77, 1500], 64)]
    shared = torch.empty(latent_workspace_bytes(), dtype=torch.uint8, device=dev)
    for ws in (None, shared):
        want = []
        for args, out in cases:
            latent_attention(out, **args)
            want.append(out.clone())
        graphs = []
        for args, out in cases:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                latent_attention(out, workspace=ws, **args)
            graphs.append(graph)
        for _ in range(3):
            for (_, out), graph in zip(cases, graphs):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(cases, want):
            assert bits_equal(out.cpu(), w.cpu())
        # fewer cached tokens, the same graph
        args, out = cases[0]
        kept = args["seq_lens"].clone()
        args["seq_lens"].copy_(torch.tensor([64, 1, 0], dtype=torch.int32))
        graphs[0].replay()
        got = out.clone()
        latent_attention(out, **args)
        torch.cuda.synchronize()
        assert bits_equal(got.cpu(), out.cpu())
        args["seq_lens"].copy_(kept)
        del graphs


def test_two_streams_at_once():
    """Calls on two streams, each with its own workspace from the allocator, give the bits of calls
    alone."""
    dev = cuda_device()
    cases = [_decode_case(43, [4000, 9], 16), _decode_case(44, [100] * 40, 128)]
    want = []
    for args, out in cases:
        latent_attention(out, **args)
        want.append(out.clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in cases]
    for (_, out) in cases:
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for (args, out), s in zip(cases, streams):
            with torch.cuda.stream(s):
                latent_attention(out, **args)
    torch.cuda.synchronize()
    for (_, out), w in zip(cases, want):
        assert bits_equal(out.cpu(), w.cpu())


def test_captured_prefill_store_and_rotation():
    dev = cuda_device()
    g = seeded(45)
    dt, t, h = torch.bfloat16, 50, 4
    cs = rope_cos_sin_cache(100, R)
    x, q = torch.randn(t, W, generator=g).to(dt).to(dev), torch.randn(t, h, 192, generator=g).to(dt).to(dev)
    pos, slots = torch.arange(t, device=dev), torch.arange(t, device=dev)
    kv = torch.randn(t, h, 256, generator=g).to(dt).to(dev)
    cu = torch.tensor([0, 20, t], dtype=torch.int32, device=dev)

    def layer(xx, qq, cache, out):
        latent_rope_and_cache(pos, qq[..., 128:], xx[:, :L], xx[:, L:], cs, cache, slots)
        latent_attention_prefill(out, qq, kv[..., :128], xx[:, L:], kv[..., 128:], cu, cu, 30, SCALE)

    want = [x.clone(), q.clone(), torch.zeros(4, 16, W, dtype=dt, device=dev), torch.zeros(t, h, 128, dtype=dt, device=dev)]
    layer(*want)
    got = [x.clone(), q.clone(), torch.zeros_like(want[2]), torch.zeros_like(want[3])]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(*got)
    got[0].copy_(x), got[1].copy_(q)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert bits_equal(a.cpu(), b.cpu())
    del graph


def test_bad_pages_and_lengths_are_reported():
    """A page id outside the cache reads as zeros, a length beyond the block table is clamped, a
    sequence with more queries than announced is left alone; each sets the error word."""
    dev = cuda_device()
    g = seeded(46)
    cache, table, rows = paged([64, 64], 16, torch.bfloat16, g, extra=0)
    table = table[:, :4].contiguous()
    ql = torch.randn(2, 16, L, generator=g).bfloat16()
    qr = torch.randn(2, 16, R, generator=g).bfloat16()
    out = torch.zeros(2, 16, L, dtype=torch.bfloat16, device=dev)
    for bad in (-1, cache.shape[0]):
        broken = table.clone()
        broken[1, 2] = bad
        latent_attention(out, ql.to(dev), qr.to(dev), cache.to(dev), torch.tensor([64, 64], dtype=torch.int32, device=dev),
                         broken.to(dev), SCALE)
        torch.cuda.synchronize()
        assert capi.read_device_error(stream()) == capi.DEVERR_INDEX_RANGE
        zeroed = rows[1].clone()
        zeroed[32:48] = 0
        ref, _, tol, _ = reference(ql, qr, [rows[0], zeroed], [0, 1, 2], SCALE)
        close(out, ref, tol)
    latent_attention(out, ql.to(dev), qr.to(dev), cache.to(dev), torch.tensor([64, 1000], dtype=torch.int32, device=dev),
                     table.to(dev), SCALE)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == capi.DEVERR_INDEX_RANGE
    ref, _, tol, _ = reference(ql, qr, rows, [0, 1, 2], SCALE)
    close(out, ref, tol)
    out.fill_(7.0)
    latent_attention(out, ql.to(dev), qr.to(dev), cache.to(dev), torch.tensor([64, 64], dtype=torch.int32, device=dev),
                     table.to(dev), SCALE, query_start_loc=torch.tensor([0, 2, 2], dtype=torch.int32, device=dev), max_query_len=1)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == capi.DEVERR_INDEX_RANGE
    assert bool((out == 7.0).all())


def test_bad_start_locations_of_prompts_are_reported():
    dev = cuda_device()
    g = seeded(47)
    q = torch.randn(40, 2, 192, generator=g).half()
    kv = torch.randn(40, 2, 256, generator=g).half()
    kr = torch.randn(40, 64, generator=g).half()
    out = torch.full((40, 2, 128), 7.0, dtype=torch.float16, device=dev)
    cu_q = torch.tensor([0, 10, 40], dtype=torch.int32, device=dev)
    cu_k = torch.tensor([0, 10, 41], dtype=torch.int32, device=dev)  # one row too many
    kvd = kv.to(dev)
    latent_attention_prefill(out, q.to(dev), kvd[..., :128], kr.to(dev), kvd[..., 128:], cu_q, cu_k, 30, SCALE)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == capi.DEVERR_INDEX_RANGE
    ref, _, tol, _ = reference_expanded(q[:10], kv[..., :128], kr, kv[..., 128:], [0, 10], [0, 10], True)
    close(out[:10], ref, tol)
    assert bool((out[10:] == 7.0).all())


def test_prompts_behind_a_falling_start_location_are_skipped():
    """They could overlap the rows before, and their number would be bounded by nothing."""
    dev = cuda_device()
    g = seeded(50)
    q = torch.randn(40, 2, 192, generator=g).half()
    kv = torch.randn(40, 2, 256, generator=g).half()
    kr = torch.randn(40, 64, generator=g).half()
    kvd = kv.to(dev)
    cu_k = torch.tensor([0, 20, 20, 40] + [40] * 40, dtype=torch.int32, device=dev)
    cu_q = torch.tensor([0, 20, 5, 25] + [40] * 40, dtype=torch.int32, device=dev)  # the last ones in a later 32
    out = torch.full((40, 2, 128), 7.0, dtype=torch.float16, device=dev)
    latent_attention_prefill(out, q.to(dev), kvd[..., :128], kr.to(dev), kvd[..., 128:], cu_q, cu_k, 30, SCALE)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == capi.DEVERR_INDEX_RANGE
    ref, _, tol, _ = reference_expanded(q[:20], kv[..., :128], kr, kv[..., 128:], [0, 20], [0, 20], True)
    close(out[:20], ref, tol)
    assert bool((out[20:] == 7.0).all())


def test_refusals():
    dev = cuda_device()
    args, out = _decode_case(48, [20, 30], 16)
    small = torch.empty(1024, dtype=torch.uint8, device=dev)
    for bad in (dict(kv_cache=args["kv_cache"][..., :512]), dict(kv_cache=args["kv_cache"].half()), dict(scale=0.0),
                dict(scale=-1.0), dict(q_rope=args["q_rope"][:1]), dict(q_latent=args["q_latent"].float()),
                dict(seq_lens=args["seq_lens"].cpu()), dict(block_table=args["block_table"][:1]), dict(workspace=small),
                dict(lse=torch.empty(2, 15, device=dev)), dict(q_latent=args["q_latent"].transpose(1, 2)),
                dict(kv_cache=torch.zeros(4, 8, W, dtype=torch.bfloat16, device=dev))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            latent_attention(out, **(args | bad))
    with pytest.raises(RuntimeError):  # rows that share memory cannot be written
        latent_attention(out[:1].expand(2, 16, L), **args)
    empty = {k: v[:0] if k in ("q_latent", "q_rope", "seq_lens", "block_table") else v for k, v in args.items()}
    latent_attention(out[:0], **empty)
    q = torch.zeros(4, 2, 192, dtype=torch.bfloat16, device=dev)
    k, r = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device=dev), torch.zeros(4, 64, dtype=torch.bfloat16, device=dev)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    base = dict(out=k.clone(), query=q, k_nope=k, k_rope=r, value=k, cu_seqlens_q=cu, cu_seqlens_k=cu, max_query_len=4, scale=0.1)
    latent_attention_prefill(**base)
    for bad in (dict(k_rope=r[:, :32]), dict(value=k[:3]), dict(query=q.half()), dict(scale=0.0), dict(cu_seqlens_k=cu[:1]),
                dict(out=q), dict(lse=torch.empty(4, 3, device=dev)), dict(k_nope=k.cpu())):
        with pytest.raises((RuntimeError, NotImplementedError)):
            latent_attention_prefill(**(base | bad))


def test_a_cache_beyond_32_bit_offsets():
    """Rows stored into and read from the far end of a 5 GB cache, as from a small one."""
    dev = cuda_device()
    g = seeded(49)
    blocks, page, t, h = 70001, 64, 150, 20
    big = torch.empty(blocks, page, W, dtype=torch.bfloat16, device=dev)
    small = torch.zeros(4, page, W, dtype=torch.bfloat16, device=dev)
    pages = torch.tensor([[blocks - 1, 0, 65536]], dtype=torch.int32)
    near = torch.tensor([[3, 0, 1]], dtype=torch.int32)
    x = torch.randn(t, W, generator=g).bfloat16().to(dev)
    ql, qr = (torch.randn(1, h, n, generator=g).bfloat16().to(dev) for n in (L, R))
    cs = rope_cos_sin_cache(t, R)
    pos = torch.arange(t)
    outs = []
    for cache, table in ((big, pages), (small, near)):
        slots = table[0, pos // page].long() * page + pos % page
        y = x.clone()
        latent_rope_and_cache(pos.to(dev), None, y[:, :L], y[:, L:], cs, cache, slots.to(dev))
        out = torch.empty_like(ql)
        latent_attention(out, ql, qr, cache, torch.tensor([t], dtype=torch.int32, device=dev), table.to(dev), SCALE)
        outs.append((out, cache[table[0].long().to(dev)].reshape(-1, W)[:t]))
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == 0
    for a, b in zip(*outs):
        assert bits_equal(a.cpu(), b.cpu())


def test_calls_without_any_key():
    """No cached token and no page, and prompts' queries without keys: zero rows, log-sums of -inf."""
    dev = cuda_device()
    dt = torch.bfloat16
    ql, qr = torch.ones(3, 5, L, dtype=dt, device=dev), torch.ones(3, 5, R, dtype=dt, device=dev)
    lens = torch.zeros(3, dtype=torch.int32, device=dev)
    for blocks, width in ((0, 0), (2, 0), (2, 4)):
        out, lse = torch.full_like(ql, 7.0), torch.full((3, 5), 7.0, device=dev)
        latent_attention(out, ql, qr, torch.full((blocks, 16, W), float("nan"), dtype=dt, device=dev), lens,
                         torch.full((3, width), -1, dtype=torch.int32, device=dev), SCALE, lse=lse)
        assert bool((out == 0).all()) and bool((lse == -torch.inf).all())
    for causal in (True, False):
        out, lse = torch.full((3, 5, 128), 7.0, dtype=dt, device=dev), torch.full((3, 5), 7.0, device=dev)
        latent_attention_prefill(out, torch.ones(3, 5, 192, dtype=dt, device=dev), torch.empty(0, 5, 128, dtype=dt, device=dev),
                                 torch.empty(0, 64, dtype=dt, device=dev), torch.empty(0, 5, 128, dtype=dt, device=dev),
                                 torch.tensor([0, 3], dtype=torch.int32, device=dev),
                                 torch.tensor([0, 0], dtype=torch.int32, device=dev), 3, SCALE, causal, lse)
        assert bool((out == 0).all()) and bool((lse == -torch.inf).all())
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == 0
