"""Measured cases of the latent-attention operators and the rotary positions that feed them.

Five operators, each as ``run`` with ``own`` false in plain torch operations and with ``own``
true as the calls a user makes of this package:

* ``table``   the cos/sin table of rotary positions, scaled for long contexts;
* ``rotary``  the rotation of query and key heads in place, interleaved or half layout, all or
  part of a head, from an fp32 table;
* ``store``   one decoder layer's latent rows on their way into the paged cache: RMS norm of
  the latent, rotation of the shared key and of the queries' rotary part, slot-mapped store;
* ``latent``  attention of new tokens over the paged latent cache (absorbed form);
* ``expand``  attention over per-head keys and values expanded from the latent, the rotary key
  shared by the heads (varlen, causal).
"""

import math

import torch

own = False

LATENT, ROPE, NOPE, VDIM = 512, 64, 128, 128
WIDTH = LATENT + ROPE
QK = NOPE + ROPE
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # a model load's table of one attention module, no scaling
        {"name": "table_4096", "op": "table", "rows": 4096, "rot": 128, "scaling": "none", "factor": 1.0, "type": "bf16"},
        # the table of a long context: yarn frequencies, 128 Ki positions and a ragged end
        {"name": "table_yarn_131075", "op": "table", "rows": 131075, "rot": 64, "scaling": "yarn", "factor": 40.0,
         "type": "f32"},
        # a small decode batch, half of each head rotated (grouped-query layer, 32/8 heads of 128)
        {"name": "rotary_half_7", "op": "rotary", "tokens": 7, "heads": 32, "kv_heads": 8, "head": 128, "rot": 64,
         "lead": 0, "layout": "half", "type": "f16"},
        # a prefill batch of a latent layer: the last 64 of each query head's 192, and the shared key
        {"name": "rotary_interleaved_4099", "op": "rotary", "tokens": 4099, "heads": 128, "kv_heads": 1, "head": 64,
         "rot": 64, "lead": 128, "layout": "interleaved", "type": "bf16"},
        # one decode token of a tensor-parallel shard: latency
        {"name": "store_1", "op": "store", "tokens": 1, "heads": 8, "page": 64, "layout": "interleaved", "type": "bf16"},
        # a prefill batch, every head on this GPU
        {"name": "store_8191", "op": "store", "tokens": 8191, "heads": 128, "page": 16, "layout": "half", "type": "f16"},
        # one sequence on a tensor-parallel shard: few rows, the context split over the GPU
        {"name": "latent_decode_1", "op": "latent", "seqs": 1, "heads": 16, "ctx": 2047, "query": 1, "ragged": False,
         "page": 16, "type": "bf16"},
        # a serving batch on a tensor-parallel shard, contexts of every length
        {"name": "latent_decode_ragged", "op": "latent", "seqs": 96, "heads": 16, "ctx": 8192, "query": 1,
         "ragged": True, "page": 64, "type": "bf16"},
        # a serving batch with every head on this GPU, long contexts
        {"name": "latent_decode_heads", "op": "latent", "seqs": 32, "heads": 128, "ctx": 16384, "query": 1,
         "ragged": False, "page": 64, "type": "bf16"},
        # chunks of new tokens over their cached contexts, odd head count
        {"name": "latent_chunk", "op": "latent", "seqs": 6, "heads": 20, "ctx": 5001, "query": 97, "ragged": True,
         "page": 32, "type": "f16"},
        # short prompts of a mixed batch
        {"name": "expand_ragged", "op": "expand", "seqs": 9, "heads": 10, "tokens": 333, "ragged": True, "past": 0,
         "type": "f16"},
        # one long prompt on a tensor-parallel shard
        {"name": "expand_long", "op": "expand", "seqs": 1, "heads": 32, "tokens": 8192, "ragged": False, "past": 0,
         "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["table", "rotary", "store", "latent", "latent", "latent", "expand", "expand"])
    half = rng.choice(["bf16", "f16"])
    if op == "table":
        return {"op": op, "rows": _log(rng, 1, 131000), "rot": 2 * rng.randint(8, 64),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "factor": round(rng.uniform(1.0, 40.0), 3),
                "type": rng.choice(["bf16", "f16", "f32"])}
    if op == "rotary":
        layout = rng.choice(["half", "interleaved"])
        heads, tokens = rng.randint(1, 128), _log(rng, 1, 4000)
        if rng.random() < 0.5:
            return {"op": op, "tokens": tokens, "heads": heads, "kv_heads": 1, "head": ROPE, "rot": ROPE, "lead": NOPE,
                    "layout": layout, "type": half}
        head = rng.choice([64, 80, 96, 128])
        return {"op": op, "tokens": tokens, "heads": min(heads, 32), "kv_heads": rng.choice([1, 2, 8]), "head": head,
                "rot": 2 * rng.randint(4, head // 2), "lead": 0, "layout": layout, "type": rng.choice([half, "f32"])}
    if op == "store":
        return {"op": op, "tokens": _log(rng, 1, 8000), "heads": rng.randint(1, 128), "page": rng.choice([16, 32, 64, 128]),
                "layout": rng.choice(["half", "interleaved"]), "type": half}
    if op == "latent":
        heads = rng.choice([1, 7, 8, 16, 20, 32, 40, 64, 96, 128, rng.randint(1, 128)])
        ctx = _log(rng, 1, 16000)
        query = 1 if rng.random() < 0.6 else _log(rng, 2, 128)
        query = max(1, min(query, ctx, 4096 // heads))
        most = min(96, (32 * 16384) // ctx, max(1, 120_000_000 // (heads * query * ctx)))
        return {"op": op, "seqs": _log(rng, 1, max(1, most)), "heads": heads, "ctx": ctx, "query": query,
                "ragged": rng.random() < 0.7, "page": rng.choice([16, 32, 64, 128]), "type": half}
    heads, tokens = rng.choice([1, 5, 8, 10, 32]), _log(rng, 1, 4000)
    past = 0 if rng.random() < 0.6 else _log(rng, 1, 4000)
    most = max(1, min(500_000_000 // (heads * tokens * (tokens + past)), 1_000_000 // (heads * (tokens + past))))
    return {"op": op, "seqs": _log(rng, 1, min(most, 32)), "heads": heads, "tokens": tokens,
            "ragged": rng.random() < 0.7, "past": past, "type": half}


def _spread(n, most, least=1):
    """n whole lengths between least and most, the first one most: the same for every seed."""
    return [most if i == 0 else least + int((most - least + 1) * ((0.618034 * i) % 1.0)) for i in range(n)]


def _lengths(case):
    """(query tokens, key tokens) of each sequence."""
    n = case["seqs"]
    if case["op"] == "latent":
        ctx = _spread(n, case["ctx"]) if case["ragged"] else [case["ctx"]] * n
        q = _spread(n, case["query"]) if case["ragged"] else [case["query"]] * n
        return [min(a, b) for a, b in zip(q, ctx)], ctx
    q = _spread(n, case["tokens"]) if case["ragged"] else [case["tokens"]] * n
    past = _spread(n, case["past"], 0) if case["ragged"] and case["past"] else [case["past"]] * n
    return q, [a + b for a, b in zip(q, past)]


def _starts(lengths, dev):
    return torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)


def _frequencies64(rot, base, scaling, factor, divisors):
    """The rotary frequencies in 64 bits (on the divisors' device)."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=divisors.device)
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = torch.exp(i * (-2.0 / rot * math.log(base)))
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        lo = max(math.floor(rot * math.log(4096 / (32.0 * 2 * math.pi)) / (2 * math.log(base))), 0)
        hi = min(math.ceil(rot * math.log(4096 / (1.0 * 2 * math.pi)) / (2 * math.log(base))), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        f = f / factor * ramp + f * (1.0 - ramp)
    return f / divisors.double()


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = TYPES[case["type"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)

    s = {"case": case}
    if case["op"] == "table":
        s["base"] = 10000.0 + float(seed % 997)
        s["divisors"] = 1.0 + torch.rand(case["rot"] // 2, generator=g, device=dev)
        return s
    if case["op"] in ("rotary", "store"):
        t, h = case["tokens"], case["heads"]
        rot = case["rot"] if case["op"] == "rotary" else ROPE
        freq = _frequencies64(rot, 10000.0, "none", 1.0, torch.ones(rot // 2, device=dev))
        angle = torch.arange(32768, dtype=torch.float64, device=dev)[:, None] * freq
        s["cos_sin"] = torch.cat((angle.cos(), angle.sin()), dim=-1).float()
        s["positions"] = torch.randint(0, 32768, (t,), generator=g, device=dev)
        if case["op"] == "rotary":
            s["query"] = normal(t, h, case["lead"] + case["head"])
            s["key"] = normal(t, case["kv_heads"], case["head"])
            return s
        # the layer's projections: queries [t, h, 192], and one row of latent and shared key
        s["query"] = normal(t, h, QK)
        row = normal(t, WIDTH)
        s["latent"], s["key"] = row[:, :LATENT], row[:, LATENT:]
        s["weight"] = normal(LATENT, std=0.2) + 1.0
        blocks = -(-t // case["page"]) + 3
        slots = torch.randperm(blocks * case["page"], generator=g, device=dev)[:t]
        s["slots"] = torch.where(torch.arange(t, device=dev) % 19 == 18, -1, slots)  # every 19th a padded row
        s["cache"] = torch.zeros(blocks, case["page"], WIDTH, dtype=dt, device=dev)
        s["normed"] = torch.zeros(t, LATENT, dtype=dt, device=dev)
        return s
    q_len, k_len = _lengths(case)
    h, t = case["heads"], sum(q_len)
    s["scale"] = QK ** -0.5
    s["max_query"], s["max_ctx"] = max(q_len), max(k_len)
    s["cu_q"], s["cu_k"] = _starts(q_len, dev), _starts(k_len, dev)
    s["q_lens"] = torch.tensor(q_len, dtype=torch.int32, device=dev)
    s["k_lens"] = torch.tensor(k_len, dtype=torch.int32, device=dev)
    s["lse"] = torch.zeros(t, h, dtype=torch.float32, device=dev)
    if case["op"] == "latent":
        page = case["page"]
        s["q_latent"], s["q_rope"] = normal(t, h, LATENT), normal(t, h, ROPE)
        pages = [-(-k // page) for k in k_len]
        blocks = sum(pages) + 5
        order = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
        table = torch.zeros(len(q_len), max(pages), dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(pages):
            table[b, :n] = order[at : at + n]
            at += n
        s["table"], s["cache"] = table, normal(blocks, page, WIDTH)
        s["out"] = torch.zeros(t, h, LATENT, dtype=dt, device=dev)
        return s
    keys = sum(k_len)
    s["query"] = normal(t, h, QK)
    kv = normal(keys, h, NOPE + VDIM)  # the up-projection's output: each head's key part, then its value
    s["k_nope"], s["value"] = kv[..., :NOPE], kv[..., NOPE:]
    s["k_rope"] = normal(keys, ROPE)
    s["out"] = torch.zeros(t, h, VDIM, dtype=dt, device=dev)
    return s


# ---- the plain forms -------------------------------------------------------------------


def _rotated(x, cos, sin, interleaved):
    """x [t, heads, rot] rotated in 32 bits; cos/sin [t, rot / 2]."""
    x, c, s = x.float(), cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1)


def _softmax_product(q, k, v, visible, scale):
    """q [b, h, i, d], k [b, h or 1, j, d], v [b, h or 1, j, e], visible [b, 1, i, j], in 32 bits:
    the attention's output [b, h, i, e] and the natural log of the sums [b, h, i]."""
    x = torch.where(visible, q @ k.transpose(-1, -2) * scale, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, p @ v / total, 0.0)
    return o, (m + torch.log(total)).squeeze(-1)


def _rows(starts, lengths, most):
    """Row numbers [b, most] of each sequence's tokens, and which of them there are."""
    i = torch.arange(most, device=starts.device)
    there = i < lengths[:, None]
    return torch.where(there, starts[:-1, None] + i, 0).long(), there


def _visible(s, there):
    j = torch.arange(s["max_ctx"], device=there.device)
    i = torch.arange(s["max_query"], device=there.device)
    last = (s["k_lens"] - s["q_lens"])[:, None] + i  # the position of each new token
    return ((j <= last[..., None]) & there[..., None])[:, None]


def _plain(s):
    case = s["case"]
    dt = TYPES[case["type"]]
    if case["op"] == "table":
        f = _frequencies64(case["rot"], s["base"], case["scaling"], case["factor"], s["divisors"])
        a = torch.arange(case["rows"], dtype=torch.float64, device=f.device)[:, None] * f
        return torch.cat((a.cos(), a.sin()), dim=-1).to(dt)
    if case["op"] == "rotary":
        cos, sin = s["cos_sin"][s["positions"]].chunk(2, dim=-1)
        n, inter, lead = case["rot"], case["layout"] == "interleaved", case["lead"]
        s["query"][..., lead : lead + n] = _rotated(s["query"][..., lead : lead + n], cos, sin, inter).to(dt)
        s["key"][..., :n] = _rotated(s["key"][..., :n], cos, sin, inter).to(dt)
        return [s["query"], s["key"]]
    if case["op"] == "store":
        cos, sin = s["cos_sin"][s["positions"]].chunk(2, dim=-1)
        inter = case["layout"] == "interleaved"
        x = s["latent"].float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
        s["normed"].copy_(x)
        s["query"][..., NOPE:] = _rotated(s["query"][..., NOPE:], cos, sin, inter).to(dt)
        s["key"].copy_(_rotated(s["key"][:, None], cos, sin, inter)[:, 0])
        row = torch.cat((s["normed"], s["key"]), dim=-1)
        kept = s["slots"] >= 0
        s["cache"].view(-1, WIDTH)[s["slots"][kept]] = row[kept]
        return [s["cache"], s["normed"], s["query"], s["key"]]
    at, there = _rows(s["cu_q"], s["q_lens"], s["max_query"])
    if case["op"] == "latent":
        j = torch.arange(s["max_ctx"], device=at.device)
        page = case["page"]
        inside = j < s["k_lens"][:, None]
        slot = torch.where(inside, s["table"][:, j // page].long() * page + j % page, 0)
        kv = torch.where(inside[..., None], s["cache"].view(-1, WIDTH)[slot].float(), 0.0)[:, None]
        q = torch.cat((s["q_latent"][at], s["q_rope"][at]), dim=-1).float()
        v = kv[..., :LATENT]
    else:
        rows, inside = _rows(s["cu_k"], s["k_lens"], s["max_ctx"])
        rope = s["k_rope"][rows][:, :, None].expand(-1, -1, case["heads"], -1)
        kv = torch.cat((s["k_nope"][rows], rope), dim=-1).float().transpose(1, 2)
        q, v = s["query"][at].float(), s["value"][rows].float().transpose(1, 2)
    if case["op"] == "latent":
        # every head of a token reads the same keys: one product over all rows of a sequence
        b, i, h, d = q.shape
        o, lse = _softmax_product(q.reshape(b, 1, i * h, d), kv, v,
                                  _visible(s, there).repeat_interleave(h, dim=2), s["scale"])
        o, lse = o.reshape(b, i, h, -1), lse.reshape(b, i, h)
    else:
        o, lse = _softmax_product(q.transpose(1, 2), kv, v, _visible(s, there), s["scale"])
        o, lse = o.transpose(1, 2), lse.transpose(1, 2)
    s["out"][at[there]] = o[there].to(dt)
    s["lse"][at[there]] = lse[there]
    return [s["out"], s["lse"]]


# ---- the package's calls ---------------------------------------------------------------


def _package():
    import sys

    if "vllm-nt_b200" not in sys.path:
        sys.path.insert(1, "vllm-nt_b200")
    from vllm_nt._ntops import torch as package

    return package


def _own(s):
    case = s["case"]
    op = _package()
    if case["op"] == "table":
        return op.rope_cos_sin_cache(case["rows"], case["rot"], s["base"], scaling=case["scaling"], factor=case["factor"],
                                     original_max_position=4096, magnitude=1.0, freq_divisors=s["divisors"],
                                     dtype=TYPES[case["type"]], device="cuda")
    if case["op"] == "rotary":
        op.rotary_embedding(s["positions"], s["query"][..., case["lead"] :], s["key"], case["head"], s["cos_sin"],
                            case["rot"], interleaved=case["layout"] == "interleaved")
        return [s["query"], s["key"]]
    if case["op"] == "store":
        op.latent_rope_and_cache(s["positions"], s["query"][..., NOPE:], s["latent"], s["key"], s["cos_sin"],
                                 s["cache"], s["slots"], norm_weight=s["weight"], eps=EPS, latent_out=s["normed"],
                                 interleaved=case["layout"] == "interleaved")
        return [s["cache"], s["normed"], s["query"], s["key"]]
    if case["op"] == "latent":
        op.latent_attention(s["out"], s["q_latent"], s["q_rope"], s["cache"], s["k_lens"], s["table"], s["scale"],
                            query_start_loc=s["cu_q"], max_query_len=s["max_query"], max_seq_len=s["max_ctx"],
                            lse=s["lse"])
    else:
        op.latent_attention_prefill(s["out"], s["query"], s["k_nope"], s["k_rope"], s["value"], s["cu_q"], s["cu_k"],
                                    s["max_query"], s["scale"], causal=True, lse=s["lse"])
    return [s["out"], s["lse"]]


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["type"]]
    if case["op"] == "table":
        n = case["rows"] * case["rot"]
        return {"bytes": n * size, "flops": 2 * n}
    if case["op"] == "rotary":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rot"]
        return {"bytes": 2 * n * size + case["tokens"] * (case["rot"] * 4 + 8), "flops": 3 * n}
    if case["op"] == "store":
        t = case["tokens"]
        n = t * (case["heads"] + 1) * ROPE
        stored = t - t // 19
        return {"bytes": size * (2 * n + 2 * t * LATENT + stored * WIDTH + LATENT) + t * (ROPE * 4 + 16),
                "flops": 3 * n + 4 * t * LATENT}
    q_len, k_len = _lengths(case)
    h, t, keys = case["heads"], sum(q_len), sum(k_len)
    pairs = h * sum(q * k - q * (q - 1) // 2 for q, k in zip(q_len, k_len))
    if case["op"] == "latent":
        return {"bytes": size * (keys * WIDTH + t * h * (WIDTH + LATENT)) + 4 * t * h,
                "flops": 2 * pairs * (WIDTH + LATENT)}
    return {"bytes": size * (keys * (h * (NOPE + VDIM) + ROPE) + t * h * (QK + VDIM)) + 4 * t * h,
            "flops": 2 * pairs * (QK + VDIM)}


# ---- the definitions in 64 bits --------------------------------------------------------


def _turn64(x, cos_sin, positions, layout):
    """Each pair (a, b) of x's last dimension as the complex number a + ib times e^(i angle)."""
    n = x.shape[-1]
    w = torch.complex(cos_sin[positions, : n // 2].double(), cos_sin[positions, n // 2 :].double())[:, None]
    x = x.double()
    if layout == "interleaved":
        z = torch.view_as_complex(x.unflatten(-1, (n // 2, 2)).contiguous()) * w
        return torch.view_as_real(z).flatten(-2)
    z = torch.complex(x[..., : n // 2].contiguous(), x[..., n // 2 :].contiguous()) * w
    return torch.cat((z.real, z.imag), dim=-1)


def _attend64(q, k, v, scale):
    """One head's q [i, d] over k [j, d], v [j, e], the queries last in the context."""
    i, j = q.shape[0], k.shape[0]
    x = (q @ k.T) * scale
    x.masked_fill_(torch.ones(i, j, dtype=torch.bool, device=q.device).triu_(j - i + 1), -math.inf)
    lse = torch.logsumexp(x, dim=-1)
    return x.sub_(lse[:, None]).exp_() @ v, lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "table":
        d, base, f = case["rot"], s["base"], case["factor"]
        rows = torch.arange(case["rows"], dtype=torch.float64, device="cuda")
        wide = []
        for i in range(d // 2):
            b = base * f ** (d / (d - 2)) if case["scaling"] == "ntk" and d > 2 else base
            w = b ** (-2 * i / d)
            if case["scaling"] == "linear":
                w /= f
            if case["scaling"] == "yarn":
                at = [d * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
                lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
                share = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
                w = w * (1 - share) + w / f * share
            wide.append(rows * (w / float(s["divisors"][i])))
        angle = torch.stack(wide, dim=-1)
        return torch.cat((torch.cos(angle), torch.sin(angle)), dim=-1)
    if case["op"] == "rotary":
        q, k, lead, n = s["query"].double(), s["key"].double(), case["lead"], case["rot"]
        q[..., lead : lead + n] = _turn64(q[..., lead : lead + n], s["cos_sin"], s["positions"], case["layout"])
        k[..., :n] = _turn64(k[..., :n], s["cos_sin"], s["positions"], case["layout"])
        return [q, k]
    if case["op"] == "store":
        x = s["latent"].double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / LATENT + EPS).sqrt() * s["weight"].double()
        q = s["query"].double()
        q[..., NOPE:] = _turn64(q[..., NOPE:], s["cos_sin"], s["positions"], case["layout"])
        k = _turn64(s["key"][:, None], s["cos_sin"], s["positions"], case["layout"])[:, 0]
        cache = s["cache"].double()
        kept = torch.nonzero(s["slots"] >= 0).flatten()
        slot = s["slots"][kept]
        cache[slot // case["page"], slot % case["page"]] = torch.cat((x, k), dim=-1)[kept]
        return [cache, x, q, k]
    q_len, k_len = _lengths(case)
    out, lse = s["out"].double(), s["lse"].double()
    q0 = k0 = 0
    for b, (nq, nk) in enumerate(zip(q_len, k_len)):
        if case["op"] == "latent":
            kv = s["cache"][s["table"][b, : -(-nk // case["page"])].long()].flatten(0, 1)[:nk].double()
        for h in range(case["heads"]):
            if case["op"] == "latent" and nq == 1:  # all heads of the token at once: they see the same keys
                q = torch.cat((s["q_latent"][q0], s["q_rope"][q0]), dim=-1).double()
                x = (q @ kv.T) * s["scale"]
                lse[q0] = torch.logsumexp(x, dim=-1)
                out[q0] = torch.softmax(x, dim=-1) @ kv[:, :LATENT]
                break
            if case["op"] == "latent":
                q = torch.cat((s["q_latent"][q0 : q0 + nq, h], s["q_rope"][q0 : q0 + nq, h]), dim=-1).double()
                k, v = kv, kv[:, :LATENT]
            else:
                q = s["query"][q0 : q0 + nq, h].double()
                k = torch.cat((s["k_nope"][k0 : k0 + nk, h], s["k_rope"][k0 : k0 + nk]), dim=-1).double()
                v = s["value"][k0 : k0 + nk, h].double()
            out[q0 : q0 + nq, h], lse[q0 : q0 + nq, h] = _attend64(q, k, v, s["scale"])
        q0, k0 = q0 + nq, k0 + nk
    return [out, lse]
