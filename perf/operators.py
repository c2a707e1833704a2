"""The attention operators of a decoder layer, as cases that can be timed and compared.

Between the q|k|v matmul and the o matmul a layer does three things (one operator each):

* ``norm_rope``: RMSNorm of every query and key head over its head_dim, times the norm weight, then the
  position rotation of the first ``rotary`` elements (pairs (i, i + rotary / 2)), for queries and keys that
  stay in plain [tokens, heads, head_dim] tensors;
* ``append``: the same on the tokens of several sequences at once, where the keys go to the pages of a paged
  cache, beside the values (RMSNorm without a weight);
* ``attention``: attention of the new tokens over the paged cache, causal, with an optional sliding window,
  several query heads to a key/value head; a prompt's chunk, or one token for each sequence.

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits (the angles in 64).
"""
import math

import torch

own = False

EPS = 1e-6


# ---- cases ---------------------------------------------------------------------------------------------
# Lengths of a batch are texts ("1,15,256"): q_lens the new tokens of each sequence, kv_lens its tokens in
# the cache with the new ones. Heads: 16 query / 8 key heads of 256 are a sliding-window layer's, 16 / 1 of
# 512 a full-attention layer's (whose key projection is the value too), 2 / 1 of 256 what one of eight
# tensor-parallel ranks has.

def listed():
    return [
        # one decoded token: what counts is the latency of the launch
        {"name": "norm_rope_one_token", "op": "norm_rope", "tokens": 1, "q_heads": 16, "kv_heads": 8,
         "head_dim": 256, "rotary": 256, "base": 10000.0, "first": 16383},
        # the last 2048-token chunk of a 16384-token prompt
        {"name": "norm_rope_chunk", "op": "norm_rope", "tokens": 2048, "q_heads": 16, "kv_heads": 8,
         "head_dim": 256, "rotary": 256, "base": 10000.0, "first": 14336},
        # one token for each of 24 sequences of a serving batch
        {"name": "append_decode_24", "op": "append", "q_lens": ",".join(["1"] * 24),
         "kv_lens": ",".join(str(17 + 41 * i) for i in range(24)), "q_heads": 16, "kv_heads": 8, "head_dim": 256,
         "rotary": 256, "base": 10000.0, "page": 16, "shared_kv": False},
        # the last chunk of a long prompt in a full-attention layer: the raw key is the value too
        {"name": "append_chunk_512", "op": "append", "q_lens": "2048", "kv_lens": "16384", "q_heads": 16,
         "kv_heads": 1, "head_dim": 512, "rotary": 128, "base": 1000000.0, "page": 64, "shared_kv": True},
        # a mixed step: prompts of several lengths beside single tokens
        {"name": "append_ragged", "op": "append", "q_lens": "1,15,256,7,700,33", "kv_lens": "911,15,1280,4096,700,2081",
         "q_heads": 16, "kv_heads": 8, "head_dim": 256, "rotary": 256, "base": 10000.0, "page": 32,
         "shared_kv": False},
        # the smallest call: one token of one sequence, sliding window
        {"name": "decode_window_1", "op": "attention", "q_lens": "1", "kv_lens": "5001", "q_heads": 16, "kv_heads": 8,
         "head_dim": 256, "page": 16, "window": 1024, "scale": 0.0625},
        # a serving batch of ragged contexts up to 16384 tokens
        {"name": "decode_batch_16", "op": "attention", "q_lens": ",".join(["1"] * 16),
         "kv_lens": "16384,129,9000,4097,1,2500,12345,640,777,3333,8192,64,1023,5120,257,6001", "q_heads": 16,
         "kv_heads": 8, "head_dim": 256, "page": 16, "window": 0, "scale": 0.0625},
        # one token over a whole long prompt, full-attention layer, scores without a scale (peaked)
        {"name": "decode_full_512", "op": "attention", "q_lens": "1", "kv_lens": "16384", "q_heads": 16, "kv_heads": 1,
         "head_dim": 512, "page": 64, "window": 0, "scale": 1.0},
        # drafted tokens verified for four sequences at once
        {"name": "verify_8x4", "op": "attention", "q_lens": "8,8,8,8", "kv_lens": "2049,1100,8,4000", "q_heads": 16,
         "kv_heads": 8, "head_dim": 256, "page": 32, "window": 1024, "scale": 0.0625},
        # a prompt's last chunk in a sliding-window layer
        {"name": "chunk_window", "op": "attention", "q_lens": "2048", "kv_lens": "16384", "q_heads": 16, "kv_heads": 8,
         "head_dim": 256, "page": 64, "window": 1024, "scale": 0.0625},
        # the same in a full-attention layer: the largest call
        {"name": "chunk_full_512", "op": "attention", "q_lens": "2048", "kv_lens": "16384", "q_heads": 16,
         "kv_heads": 1, "head_dim": 512, "page": 64, "window": 0, "scale": 0.04419417382415922},
        # prompts of several lengths beside single tokens, no window
        {"name": "chunk_ragged", "op": "attention", "q_lens": "256,1,700,33,1,512", "kv_lens": "256,4097,2748,33,901,1536",
         "q_heads": 16, "kv_heads": 8, "head_dim": 256, "page": 16, "window": 0, "scale": 0.0625},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    hq, hk, d = rng.choice([(16, 8, 256), (16, 8, 256), (16, 1, 512), (2, 1, 256), (8, 4, 256), (32, 8, 128), (12, 4, 64)])
    op = rng.choice(["norm_rope", "append", "attention", "attention", "attention"])
    c = {"op": op, "q_heads": hq, "kv_heads": hk, "head_dim": d}
    if op == "norm_rope":
        c.update(tokens=_log(rng, 1, 2048), rotary=rng.choice([d, d // 2, d // 4]), base=rng.choice([10000.0, 1000000.0]),
                 first=rng.randrange(0, 200000))
        return c
    form = rng.choice(["tokens", "verify", "mixed", "chunk"])
    if form == "tokens":
        q = [1] * _log(rng, 1, 32)
    elif form == "verify":
        q = [rng.randrange(2, 16)] * _log(rng, 1, 8)
    elif form == "mixed":
        q = [_log(rng, 1, 500) for _ in range(rng.randrange(2, 7))]
    else:
        q = [_log(rng, 64, 2048)]
    most = 16384 if op == "attention" else 4096
    # the padded score matrix of the plain form stays below the largest listed one's
    room = 2048 * 16384 * 16 // (len(q) * max(q) * hq)
    kv = [n + (rng.randrange(0, 3) if rng.random() < 0.2 else _log(rng, 1, most) - 1) for n in q]
    total = 65536 if op == "attention" else 16384
    kv = [max(n, min(k, room, total // len(q))) for n, k in zip(q, kv)]
    c.update(q_lens=",".join(map(str, q)), kv_lens=",".join(map(str, kv)), page=rng.choice([16, 32, 64, 128]))
    if op == "append":
        c.update(rotary=rng.choice([d, d // 2]), base=rng.choice([10000.0, 1000000.0]), shared_kv=hk == 1 and d == 512)
    else:
        c.update(window=rng.choice([0, 0, 1024, 1024, 517]), scale=rng.choice([d ** -0.5, d ** -0.5, 1.0]))
    return c


def _lens(text):
    return [int(t) for t in text.split(",")]


# ---- inputs --------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, mean=0.0, std=1.0):
    """bf16 N(mean, std)."""
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(torch.bfloat16)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _generator(seed)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    s = {"case": case}
    if case["op"] == "norm_rope":
        n = case["tokens"]
        row = _normal(g, n, (hq + 2 * hk) * d, std=1.7)          # a row of the q|k|v matmul
        s["q"] = row[:, : hq * d].unflatten(1, (hq, d))
        s["k"] = row[:, hq * d: (hq + hk) * d].unflatten(1, (hk, d))
        s["positions"] = torch.arange(case["first"], case["first"] + n, dtype=torch.int32, device="cuda")
    else:
        q_lens, kv_lens, page = _lens(case["q_lens"]), _lens(case["kv_lens"]), case["page"]
        n = sum(q_lens)
        used = [-(-k // page) for k in kv_lens]
        pages = sum(used) + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(used), max(used)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, u in enumerate(used):
            table[b, :u] = order[at:at + u]
            at += u
        s["block_table"] = table
        s["q_offsets"] = _int32([sum(q_lens[:b]) for b in range(len(q_lens) + 1)])
        s["kv_lens"] = _int32(kv_lens)
        s["max_q"], s["max_kv"] = max(q_lens), max(kv_lens)
        s["k_pages"] = _normal(g, pages, hk, page, d)
        s["v_pages"] = _normal(g, pages, hk, page, d)
        if case["op"] == "append":
            row = _normal(g, n, (hq + (hk if case["shared_kv"] else 2 * hk)) * d, std=1.7)
            s["q"] = row[:, : hq * d].unflatten(1, (hq, d))
            s["k"] = row[:, hq * d: (hq + hk) * d].unflatten(1, (hk, d))
            s["v"] = s["k"] if case["shared_kv"] else row[:, (hq + hk) * d:].unflatten(1, (hk, d))
        else:
            s["q"] = _normal(g, n, hq, d)
    if case["op"] != "attention":
        s["q_weight"] = _normal(g, d, mean=1.0, std=0.1)
        s["k_weight"] = _normal(g, d, mean=1.0, std=0.1)
    if own:
        from helios_b200 import attention as A
        if case["op"] != "attention":
            s["rope"] = A.Rope(d, base=case["base"], rotary_dim=case["rotary"])
        else:
            s["attend"] = A.PagedAttention(hq, hk, d)
        if case["op"] != "norm_rope":
            s["cache"] = A.PagedKVCache(s["k_pages"], s["v_pages"])
            s["batch"] = A.PagedBatch(s["q_offsets"], s["kv_lens"], s["block_table"], max_q=s["max_q"], max_kv=s["max_kv"])
    return s


# ---- one pass ------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        from helios_b200 import attention as A
        if c["op"] == "norm_rope":
            q, k = A.qk_norm_rope(s["q"], s["k"], s["positions"], s["rope"], s["q_weight"], s["k_weight"], eps=EPS)
            return {"q": q, "k": k}
        if c["op"] == "append":
            q = A.kv_append(s["q"], s["k"], s["v"], s["cache"], s["batch"], s["rope"], s["q_weight"], s["k_weight"],
                            eps=EPS)
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        return s["attend"](s["q"], s["cache"], s["batch"], scale=c["scale"], window=c["window"])
    if c["op"] == "norm_rope":
        cos, sin = _angles(s["positions"], c["rotary"], c["base"])
        return {"q": _rotate(_norm(s["q"], s["q_weight"]), cos, sin).to(torch.bfloat16),
                "k": _rotate(_norm(s["k"], s["k_weight"]), cos, sin).to(torch.bfloat16)}
    seq, pos = _tokens(s)
    if c["op"] == "append":
        cos, sin = _angles(pos, c["rotary"], c["base"])
        page, slot = s["block_table"][seq, pos // c["page"]].long(), pos % c["page"]
        s["k_pages"][page, :, slot] = _rotate(_norm(s["k"], s["k_weight"]), cos, sin).to(torch.bfloat16)
        s["v_pages"][page, :, slot] = _norm(s["v"], None).to(torch.bfloat16)
        return {"q": _rotate(_norm(s["q"], s["q_weight"]), cos, sin).to(torch.bfloat16),
                "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return _attention(s, seq, pos)


def _tokens(s):
    """(sequence, position) of every new token: a sequence's new tokens are its last ones."""
    at = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.bucketize(at, s["q_offsets"][1:].long(), right=True)
    first = (s["kv_lens"] - (s["q_offsets"][1:] - s["q_offsets"][:-1])).long()
    return seq, first[seq] + at - s["q_offsets"].long()[seq]


def _norm(x, weight):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x if weight is None else x * weight.float()


def _angles(positions, rotary, base):
    """cos and sin [tokens, 1, rotary / 2]; the angles in 64 bits, as positions reach far."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
    a = positions.double()[:, None, None] * base ** (-2.0 * i / rotary)
    return torch.cos(a).float(), torch.sin(a).float()


def _rotate(x, cos, sin):
    h = cos.shape[-1]
    a, b, rest = x[..., :h], x[..., h: 2 * h], x[..., 2 * h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _attention(s, seq, pos):
    c = s["case"]
    hk, d = c["kv_heads"], c["head_dim"]
    group, batch = c["q_heads"] // hk, s["kv_lens"].shape[0]
    table = s["block_table"].clamp(min=0).long()
    at = torch.arange(table.shape[1] * c["page"], device="cuda")
    # every sequence's pages side by side: [batch, kv head, key, head_dim]
    k = s["k_pages"][table].permute(0, 2, 1, 3, 4).reshape(batch, hk, -1, d).float()
    v = s["v_pages"][table].permute(0, 2, 1, 3, 4).reshape(batch, hk, -1, d).float()
    # the queries padded to the longest sequence: [batch, kv head, query, group, head_dim]
    row = torch.arange(s["q"].shape[0], device="cuda") - s["q_offsets"].long()[seq]
    q = torch.zeros(batch, hk, s["max_q"], group, d, device="cuda")
    q[seq, :, row] = s["q"].float().unflatten(1, (hk, group))
    p = torch.full((batch, s["max_q"]), -1, dtype=torch.long, device="cuda")
    p[seq, row] = pos
    seen = (at <= p[..., None]) & (at < s["kv_lens"].long()[:, None, None])
    if c["window"]:
        seen &= at > p[..., None] - c["window"]
    scores = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (s["max_q"], group)).mul_(c["scale"])
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = scores.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = e.sum(-1, keepdim=True)
    out = (e.flatten(2, 3) @ v).unflatten(2, (s["max_q"], group)) / torch.where(total > 0, total, 1.0)
    return out[seq, :, row].flatten(1, 2).to(torch.bfloat16)


# ---- what a pass cannot do without -----------------------------------------------------------------------

def work(case):
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] != "attention":
        n = case["tokens"] if case["op"] == "norm_rope" else sum(_lens(case["q_lens"]))
        heads = hq + hk
        read, written = heads, heads
        if case["op"] == "append":
            read, written = heads + (0 if case["shared_kv"] else hk), heads + hk
        # a value is squared, summed and scaled, weighted, and rotated (two products, a sum): about 8 operations
        return {"bytes": n * (read + written) * d * 2 + 2 * d * 2 + 4 * n, "flops": 8 * n * written * d}
    pairs = keys = 0
    for q, kv in zip(_lens(case["q_lens"]), _lens(case["kv_lens"])):
        w = case["window"] or kv
        pairs += sum(min(w, p + 1) for p in range(kv - q, kv))
        keys += min(kv, w + q - 1)
    n = sum(_lens(case["q_lens"]))
    return {"bytes": 2 * keys * hk * d * 2 + 2 * n * hq * d * 2, "flops": 4 * pairs * hq * d}


# ---- the definitions in 64 bits --------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]

    def normed(x, w):
        x = x.double()
        y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + EPS)
        return y if w is None else y * w.double()

    def turned(x, where):
        """Each pair as a complex number, times exp(i * angle)."""
        r = case["rotary"]
        f = torch.tensor([case["base"] ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones_like(f)[None], where.double()[:, None] * f)[:, None]
        z = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2: r].contiguous()) * turn
        return torch.cat((z.real, z.imag, x[..., r:]), dim=-1)

    if case["op"] == "norm_rope":
        return {"q": turned(normed(s["q"], s["q_weight"]), s["positions"]),
                "k": turned(normed(s["k"], s["k_weight"]), s["positions"])}
    q_lens, kv_lens, page = _lens(case["q_lens"]), _lens(case["kv_lens"]), case["page"]
    if case["op"] == "append":
        where = torch.cat([torch.arange(k - q, k, device="cuda") for q, k in zip(q_lens, kv_lens)])
        k, v = turned(normed(s["k"], s["k_weight"]), where), normed(s["v"], None)
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        at = 0
        for b, (q, n) in enumerate(zip(q_lens, kv_lens)):
            p = torch.arange(n - q, n, device="cuda")
            rows = s["block_table"][b].long()[torch.div(p, page, rounding_mode="floor")]
            k_pages[rows, :, p % page] = k[at:at + q]
            v_pages[rows, :, p % page] = v[at:at + q]
            at += q
        return {"q": turned(normed(s["q"], s["q_weight"]), where), "k_pages": k_pages, "v_pages": v_pages}
    out = torch.zeros(sum(q_lens), hq, d, dtype=torch.float64, device="cuda")
    at = 0
    for b, (q, n) in enumerate(zip(q_lens, kv_lens)):
        mine = s["block_table"][b, : -(-n // page)].long()
        p = torch.arange(n - q, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        hidden = (j > p) | (j <= p - case["window"] if case["window"] else j < 0)
        for h in range(hq):
            kv = h // (hq // hk)
            k = s["k_pages"][mine, kv].reshape(-1, d)[:n].double()
            v = s["v_pages"][mine, kv].reshape(-1, d)[:n].double()
            x = (s["q"][at:at + q, h].double() @ k.T) * case["scale"]
            out[at:at + q, h] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v
        at += q
    return out
