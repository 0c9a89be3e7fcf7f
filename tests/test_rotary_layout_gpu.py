"""GPU parity of the rotary operators in both layouts (ntb200_rotary_embedding), their table
(ntb200_rope_cos_sin_cache) and the latent-cache store (ntb200_latent_rope_and_cache) against
their formulas in 64 bits.

Tolerances, element by element; u is half a step of the storage type (2^-8 bf16, 2^-11 fp16,
2^-24 fp32).  A rotated element is a c -+ b s with two fp32 products and a sum, each off by
2^-24 of its value: 2^-22 (|a c| + |b s|), then rounded once, u |out| (plus fp16's subnormal
half step 2^-25).  A normalised element is three fp32 products and rsqrtf of a sum of 512
squares in 16 + 5 additions: below 2^-18 of its value, then u.  A table entry is sincosf (2 ulp
of at most 1) of an angle rounded to fp32 (|r| <= pi, off by 2^-23) after an fp64 reduction."""

import math

import pytest
import torch

from _util import bits_equal, cuda_device, seeded, stream
from vllm_nt._ntops import capi
from vllm_nt._ntops.torch._ext import ops
from vllm_nt._ntops.torch import latent_rope_and_cache, rope_cos_sin_cache, rotary_embedding

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


@pytest.fixture(autouse=True)
def _clean_device_error():
    dev = cuda_device()
    torch.cuda.synchronize(dev)
    capi.read_device_error(stream())
    yield
    torch.cuda.synchronize(dev)


def table(rows, rot, dtype=torch.float32):
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * f
    return torch.cat((a.cos(), a.sin()), -1).to(dtype)


def turned(x, cs, pos, rot, interleaved):
    """x [t, heads, d] with its first rot dims rotated, and the tolerance, in 64 bits."""
    u = U[x.dtype]
    y = x.double()
    c, s = cs[pos, : rot // 2].double()[:, None], cs[pos, rot // 2 : rot].double()[:, None]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    tol = torch.zeros_like(y)
    tol[..., first] = 2.0**-22 * ((a * c).abs() + (b * s).abs())
    tol[..., second] = 2.0**-22 * ((b * c).abs() + (a * s).abs())
    tol[..., :rot] += u * y[..., :rot].abs() + (2.0**-25 if x.dtype == torch.float16 else 0.0)
    return y, tol


def close(got, ref, tol):
    err = (got.cpu().double() - ref).abs()
    assert bool((err <= tol).all()), (err - tol).max()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype,table_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                               (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                               (torch.float16, torch.float16)])
@pytest.mark.parametrize("tokens,hq,hk,head,rot", [(1, 1, 0, 64, 64), (7, 32, 8, 128, 64), (33, 5, 1, 80, 48),
                                                   (300, 20, 2, 96, 96), (5, 3, 3, 64, 10), (2, 2, 1, 512, 512),
                                                   (3, 130, 1, 64, 2)])
def test_rotation(tokens, hq, hk, head, rot, dtype, table_dtype, interleaved):
    """Whole and part heads, vector and pair-by-pair rows, one table row to hundreds.  (The half
    layout with a table of its own dtype goes to the in-place NeoX op through the Python
    entry; the C entry is called here.)"""
    dev = cuda_device()
    g = seeded(tokens + rot)
    q = torch.randn(tokens, hq, head, generator=g).to(dtype)
    k = torch.randn(tokens, hk, head, generator=g).to(dtype) if hk else None
    pos = torch.randint(0, 5000, (tokens,), generator=g)
    cs = table(5000, rot, table_dtype)
    qd, kd = q.to(dev), None if k is None else k.to(dev)
    ops().rotary_embedding(pos.to(dev), qd, kd, cs.to(dev), head, rot, interleaved)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == 0
    close(qd, *turned(q, cs, pos, rot, interleaved))
    if k is not None:
        close(kd, *turned(k, cs, pos, rot, interleaved))


@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_part_at_the_end_of_a_head(interleaved):
    """The last 64 of each head's 192 and a shared key of one projection's row, as slices; int32
    positions; what is not rotated keeps its bits."""
    dev = cuda_device()
    g = seeded(4)
    t, h = 37, 20
    q = torch.randn(t, h, 192, generator=g).bfloat16()
    row = torch.randn(t, 576, generator=g).bfloat16()
    pos = torch.randint(0, 900, (t,), generator=g)
    cs = table(900, 64)
    qd, rowd = q.to(dev), row.to(dev)
    rotary_embedding(pos.to(dev, torch.int32), qd[..., 128:], rowd[:, None, 512:], 64, cs.to(dev), interleaved=interleaved)
    torch.cuda.synchronize()
    close(qd[..., 128:], *turned(q[..., 128:], cs, pos, 64, interleaved))
    close(rowd[:, None, 512:], *turned(row[:, None, 512:], cs, pos, 64, interleaved))
    assert bits_equal(qd[..., :128].cpu(), q[..., :128]) and bits_equal(rowd[:, :512].cpu(), row[:, :512])


def test_unaligned_rows_go_pair_by_pair():
    dev = cuda_device()
    g = seeded(5)
    t, h, d = 9, 3, 64
    for interleaved, skew in ((True, 2), (False, 1)):
        wide = torch.randn(t, h, d + 6, generator=g).half()
        x = wide[..., skew : skew + d]
        pos = torch.randint(0, 50, (t,), generator=g)
        cs = table(50, d)
        wd = wide.to(dev)
        rotary_embedding(pos.to(dev), wd[..., skew : skew + d], None, d, cs.to(dev), interleaved=interleaved)
        torch.cuda.synchronize()
        close(wd[..., skew : skew + d], *turned(x, cs, pos, d, interleaved))
        assert bits_equal(wd[..., :skew].cpu(), wide[..., :skew])
        assert bits_equal(wd[..., skew + d :].cpu(), wide[..., skew + d :])
    with pytest.raises(RuntimeError, match="aligned"):  # an odd start splits every interleaved pair
        rotary_embedding(pos.to(dev), wd[..., 1 : 1 + d], None, d, cs.to(dev), interleaved=True)


def test_positions_outside_the_table_are_reported_and_left():
    dev = cuda_device()
    g = seeded(6)
    x = torch.randn(4, 2, 64, generator=g).bfloat16()
    pos = torch.tensor([3, -1, 10, 9])
    cs = table(10, 64)
    xd = x.to(dev)
    rotary_embedding(pos.to(dev), xd, None, 64, cs.to(dev), interleaved=True)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == capi.DEVERR_INDEX_RANGE
    ok = [0, 3]
    close(xd[ok], *turned(x[ok], cs, pos[ok], 64, True))
    assert bits_equal(xd[1:3].cpu(), x[1:3])


def test_rotation_refusals():
    dev = cuda_device()
    x = torch.zeros(4, 2, 64, device=dev, dtype=torch.bfloat16)
    pos = torch.zeros(4, dtype=torch.int64, device=dev)
    cs = table(10, 64).to(dev)
    for bad in (dict(rotary_dim=128), dict(rotary_dim=63), dict(positions=pos.float()), dict(cos_sin_cache=cs.half()),
                dict(cos_sin_cache=cs.cpu()), dict(positions=pos[:3]), dict(key=x.half())):
        kw = dict(positions=pos, query=x, key=None, head_size=64, cos_sin_cache=cs, interleaved=True) | bad
        with pytest.raises(RuntimeError):
            rotary_embedding(**kw)


# ---- the table ----


def frequencies(rot, base, scaling, factor, original=4096, fast=32.0, slow=1.0):
    f = []
    for i in range(rot // 2):
        b = base * factor ** (rot / (rot - 2)) if scaling == "ntk" and rot > 2 else base
        w = b ** (-2 * i / rot)
        if scaling == "linear":
            w /= factor
        if scaling == "yarn":
            at = [rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (fast, slow)]
            lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
            share = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = w * (1 - share) + w / factor * share
        f.append(w)
    return torch.tensor(f, dtype=torch.float64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
@pytest.mark.parametrize("rows,rot,first", [(1, 2, 0), (513, 64, 0), (77, 128, 1 << 20), (9, 80, (1 << 30) + 1), (3, 1026, 5)])
def test_table(rows, rot, first, scaling, dtype):
    factor, mag = 8.5, 1.25
    g = seeded(rows)
    div = 1.0 + torch.rand(rot // 2, generator=g)
    got = rope_cos_sin_cache(rows, rot, 500000.0, scaling=scaling, factor=factor, original_max_position=4096,
                             magnitude=mag, freq_divisors=div.to(cuda_device()), first_position=first, dtype=dtype)
    f = frequencies(rot, 500000.0, scaling, factor) / div.double()
    a = (first + torch.arange(rows, dtype=torch.float64))[:, None] * f
    ref = mag * torch.cat((a.cos(), a.sin()), -1)
    # fp64: a frequency is off by a few 2^-53 of it times ln(base^(..)) <= 14, the angle likewise
    tol = mag * (2.0**-22 + 2.0**-23 + 64 * 2.0**-53 * a.abs().max()) + 2 * U[dtype] * ref.abs() + 2.0**-25
    close(got, ref, tol)


def test_table_defaults_and_padded_rows():
    dev = cuda_device()
    plain = rope_cos_sin_cache(100, 64)
    close(plain, table(100, 64, torch.float64), torch.full((100, 64), 2.0**-21))
    yarn = rope_cos_sin_cache(10, 64, scaling="yarn", factor=40.0, original_max_position=4096)
    assert abs(float(yarn[0, 0]) - (0.1 * math.log(40.0) + 1.0)) < 1e-6
    wide = torch.full((100, 72), 7.0, device=dev)
    assert rope_cos_sin_cache(100, 64, out=wide) is wide
    assert bits_equal(wide[:, :64].cpu(), plain.cpu()) and bool((wide[:, 64:] == 7.0).all())
    assert rope_cos_sin_cache(0, 64).shape == (0, 64)


def test_table_refusals():
    dev = cuda_device()
    for bad in (dict(rotary_dim=63), dict(base=1.0), dict(factor=0.0), dict(factor=float("inf")), dict(scaling="other"),
                dict(scaling="yarn"), dict(scaling="yarn", original_max_position=4096, beta_fast=0.5),
                dict(first_position=-1), dict(dtype=torch.float64), dict(magnitude=float("nan")),
                dict(freq_divisors=torch.ones(31, device=dev)), dict(freq_divisors=torch.ones(32))):
        with pytest.raises((RuntimeError, ValueError)):
            rope_cos_sin_cache(**(dict(num_positions=4, rotary_dim=64) | bad))


# ---- the latent-cache store ----

EPS = 1e-6


def store_reference(latent, weight):
    x = latent.double()
    if weight is None:
        return x, torch.zeros_like(x)
    y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    return y, (U[latent.dtype] + 2.0**-18) * y.abs() + (2.0**-25 if latent.dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,page,ld,rd,normed,t32", [
    (1, 8, 64, 512, 64, True, True), (70, 20, 16, 512, 64, True, True), (300, 1, 48, 512, 64, True, False),
    (41, 128, 128, 512, 64, False, True), (9, 3, 16, 256, 32, True, True), (9, 0, 16, 1024, 256, True, True),
    (5, 2, 1, 8, 48, True, False)])
def test_latent_store(tokens, heads, page, ld, rd, normed, t32, dtype, interleaved):
    """Latent and key as columns of one projection's rows, queries as the last columns of wider
    heads, a cache with padded rows; padding slots, rows past the slot mapping, every other cache
    element and the columns that are not rotated keep their bits."""
    dev = cuda_device()
    g = seeded(tokens + heads)
    row = torch.randn(tokens, ld + rd, generator=g).to(dtype)
    q = torch.randn(tokens, heads, 128 + rd, generator=g).to(dtype)
    weight = (1.0 + 0.3 * torch.randn(ld, generator=g)).to(dtype) if normed else None
    pos = torch.randint(0, 700, (tokens,), generator=g)
    cs = table(700, rd, torch.float32 if t32 else dtype)
    blocks = -(-tokens // page) + 2
    slots = torch.randperm(blocks * page, generator=g)[: max(tokens - 2, 1)]
    slots[3::5] = -1
    cache = torch.randn(blocks, page, ld + rd + 8, generator=g).to(dtype)
    rowd, qd, cached = row.to(dev), q.to(dev), cache.to(dev)
    out = torch.full((tokens, ld), 7.0, dtype=dtype, device=dev)
    latent_rope_and_cache(pos.to(dev), qd[..., 128:] if heads else None, rowd[:, :ld], rowd[:, ld:], cs.to(dev),
                          cached[..., : ld + rd], slots.to(dev), norm_weight=None if weight is None else weight.to(dev),
                          eps=EPS, latent_out=out, interleaved=interleaved)
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == 0
    y, ytol = store_reference(row[:, :ld], weight)
    k, ktol = turned(row[:, None, ld:], cs, pos, rd, interleaved)
    close(out, y, ytol)
    close(rowd[:, None, ld:], k, ktol)
    if heads:
        close(qd[..., 128:], *turned(q[..., 128:], cs, pos, rd, interleaved))
    assert bits_equal(qd[..., :128].cpu(), q[..., :128]) and bits_equal(rowd[:, :ld].cpu(), row[:, :ld])
    want = cache.clone()
    kept = torch.nonzero(slots >= 0).flatten()
    stored = torch.cat((out.cpu(), rowd[:, ld:].cpu()), -1)  # what is cached is what is returned, bit for bit
    want[slots[kept] // page, slots[kept] % page, : ld + rd] = stored[kept]
    assert bits_equal(cached.cpu(), want)


def test_latent_store_in_place_int32_and_bad_indices():
    dev = cuda_device()
    g = seeded(8)
    row = torch.randn(6, 576, generator=g).bfloat16()
    weight = torch.ones(512).bfloat16()
    pos = torch.tensor([0, 5, 99, -3, 1, 2], dtype=torch.int32)  # two outside the table of 50
    slots = torch.tensor([0, 64, 3, 4, -1, 31], dtype=torch.int32)  # slot 64 is past the 32 there are
    cs = table(50, 64)
    rowd, cache = row.to(dev), torch.zeros(2, 16, 576, dtype=torch.bfloat16, device=dev)
    latent_rope_and_cache(pos.to(dev), None, rowd[:, :512], rowd[:, 512:], cs.to(dev), cache, slots.to(dev),
                          norm_weight=weight.to(dev), eps=EPS, latent_out=rowd[:, :512])
    torch.cuda.synchronize()
    assert capi.read_device_error(stream()) == capi.DEVERR_INDEX_RANGE
    close(rowd[:, :512], *store_reference(row[:, :512], weight))
    for t, turns in enumerate((True, True, False, False, True, True)):
        if turns:
            close(rowd[t : t + 1, None, 512:], *turned(row[t : t + 1, None, 512:], cs, pos[t : t + 1].long(), 64, True))
        else:
            assert bits_equal(rowd[t, 512:].cpu(), row[t, 512:])
    want = torch.zeros(32, 576, dtype=torch.bfloat16)
    want[[0, 3, 4, 31]] = rowd.cpu()[[0, 2, 3, 5]]
    assert bits_equal(cache.cpu().view(32, 576), want)


def test_latent_store_without_tokens_and_refusals():
    dev = cuda_device()
    bf = torch.bfloat16
    cs = table(50, 64).to(dev)
    base = dict(positions=torch.zeros(4, dtype=torch.int64, device=dev), query=torch.zeros(4, 2, 64, dtype=bf, device=dev),
                latent=torch.zeros(4, 512, dtype=bf, device=dev), key=torch.zeros(4, 64, dtype=bf, device=dev),
                cos_sin_cache=cs, kv_cache=torch.zeros(2, 16, 576, dtype=bf, device=dev),
                slot_mapping=torch.arange(4, device=dev))
    empty = {n: base[n][:0] for n in ("positions", "query", "latent", "key", "slot_mapping")}
    latent_rope_and_cache(**(base | empty))
    f32 = dict(latent=base["latent"].float(), key=base["key"].float(), query=base["query"].float(),
               kv_cache=base["kv_cache"].float())
    wide = torch.zeros(4, 600, dtype=bf, device=dev)
    for bad in (f32, dict(key=base["key"].half()), dict(kv_cache=torch.zeros(2, 16, 512, dtype=bf, device=dev)),
                dict(slot_mapping=torch.arange(5, device=dev)), dict(slot_mapping=torch.arange(4, device=dev).float()),
                dict(cos_sin_cache=cs[:, :32]), dict(latent=wide[:, 1:513]), dict(latent=wide[:, :513]),
                dict(norm_weight=torch.ones(511, dtype=bf, device=dev)), dict(query=base["query"][:3]),
                dict(latent_out=torch.zeros(4, 500, dtype=bf, device=dev)), dict(positions=base["positions"].cpu()),
                dict(cos_sin_cache=cs.half())):
        with pytest.raises((RuntimeError, NotImplementedError)):
            latent_rope_and_cache(**(base | bad))
