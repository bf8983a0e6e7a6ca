"""The 4-bit KV cache operators as measured work: RoPE + quantising append,
decode attention, both in one call, and attention of many queries a sequence.

Every case runs in two ways on the same inputs: ``own`` False computes the
operator from elementary torch operations in 32 bits (64 where a rounding
decides a code: the rotation and the quantiser), ``own`` True calls
:mod:`llamamps_b200.kernels`.

The cache: one layer's K (and V) pool is uint8 [n_pages, n_kv_heads,
page_size * 72]; a (page, head) block is page_size rows of 64 code bytes
(element 2j of the 128 in the low nibble of byte j, 2j + 1 in the high one,
code + 8) followed by page_size rows of 4 fp16 scales, one per 32 elements.
"""
import math
import random

import torch

own = False

HEAD_DIM = 128
GROUP = 32
ROW_BYTES = 72
SCALE = 0.088388  # the score scale of the framework's attention
HEADS = [(12, 2), (12, 2), (12, 2), (6, 1), (16, 2), (32, 8), (8, 8), (10, 2), (7, 1)]


# -- cases ---------------------------------------------------------------------
def listed():
    return [
        # one new token of one sequence: the append of a batch-1 decode step
        dict(name="append 1 token", op="append", batch=1, seq=1, lo=1000, hi=1000, ragged=1, hq=12, hkv=2, page=64,
             style=0),
        # one new token of each of 64 sequences at ragged positions of a long cache (a batched decode step)
        dict(name="append 64 tokens", op="append", batch=64, seq=1, lo=1, hi=32700, ragged=2, hq=12, hkv=2, page=64,
             style=1),
        # every token of 8 prompts of 2048 at once (the benchmark's prefill)
        dict(name="append 8x2048 prompt", op="append", batch=8, seq=2048, lo=2048, hi=2048, ragged=3, hq=12, hkv=2,
             page=64, style=0),
        # batch-1 decode with a short context: the latency case
        dict(name="decode 1x131", op="decode", batch=1, lo=131, hi=131, ragged=4, hq=12, hkv=2, page=64),
        # 64 sequences of ragged medium contexts, small pages
        dict(name="decode 64x1..1000", op="decode", batch=64, lo=1, hi=1000, ragged=5, hq=12, hkv=2, page=16),
        # the benchmark's long-context decode: 4 sequences at 32K
        dict(name="decode 4x32768", op="decode", batch=4, lo=32768, hi=32768, ragged=6, hq=12, hkv=2, page=64),
        # a full decode batch with long ragged contexts: the bandwidth case
        dict(name="decode 64x4100..8200", op="decode", batch=64, lo=4100, hi=8200, ragged=7, hq=12, hkv=2, page=64),
        # one decode step's attention of one sequence, rotation and append included
        dict(name="step 1x2049", op="step", batch=1, lo=2049, hi=2049, ragged=8, hq=12, hkv=2, page=64, style=0),
        # the same for a decode batch, one rank's heads of the two-way split
        dict(name="step 64x500..2100", op="step", batch=64, lo=500, hi=2100, ragged=9, hq=6, hkv=1, page=64, style=1),
        # a short odd prompt
        dict(name="prefill 1x37", op="prefill", batch=1, seq=37, lo=0, hi=0, ragged=10, hq=12, hkv=2, page=64),
        # the benchmark's prefill: 8 prompts of 2048
        dict(name="prefill 8x2048", op="prefill", batch=8, seq=2048, lo=0, hi=0, ragged=11, hq=12, hkv=2, page=64),
        # the next turn of 4 chats: ragged chunks of up to 256 tokens behind ragged cached contexts
        dict(name="extend 4x256 at 1..30000", op="prefill", batch=4, seq=256, lo=1, hi=30000, ragged=12, hq=12,
             hkv=2, page=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(work(c)["flops"] for c in listed() if c["op"] == "prefill")
    while True:
        op = rng.choice(["append", "decode", "step", "prefill"])
        hq, hkv = rng.choice(HEADS)
        c = dict(op=op, ragged=rng.randrange(1 << 20), hq=hq, hkv=hkv, page=rng.choice([16, 32, 48, 64, 64, 128]))
        if op == "append":
            c["style"] = rng.randrange(2)
            if rng.random() < 0.5:  # one token each of a decode batch
                hi = _log_int(rng, 1, 32768)
                c.update(batch=_log_int(rng, 1, 64), seq=1, lo=rng.randint(1, hi), hi=hi)
                if c["batch"] * hi * hkv > 64 * 32768 * 2:
                    continue
            else:  # whole prompts
                s = _log_int(rng, 2, 2048)
                c.update(batch=_log_int(rng, 1, 8), seq=s, lo=s, hi=s)
            if work(c)["bytes"] > 1.2e8:
                continue
        elif op in ("decode", "step"):
            hi = _log_int(rng, 1, 32768)
            c.update(batch=_log_int(rng, 1, 64), lo=rng.randint(1, hi), hi=hi)
            if op == "step":
                c["style"] = rng.randrange(2)
            if c["batch"] * hi * hkv > 64 * 8200 * 2:
                continue
        else:
            hi = rng.choice([0, _log_int(rng, 1, 30000)])
            c.update(batch=_log_int(rng, 1, 8), seq=_log_int(rng, 1, 2048), lo=rng.randint(0, hi), hi=hi)
            if work(c)["flops"] > most or c["batch"] * c["seq"] * (hi + c["seq"]) * hq > 8 * 2048 * 2048 * 12:
                continue
        return c


def _spread(case, lo, hi, n, salt=0):
    """n whole numbers of [lo, hi], hi among them, fixed by the case."""
    r = random.Random(1000 * case["ragged"] + salt)
    v = [hi] + [r.randint(lo, hi) for _ in range(n - 1)]
    r.shuffle(v)
    return v


def _plan(case):
    """Per sequence: cached positions before the call's own, new tokens of the call."""
    B = case["batch"]
    if case["op"] == "append":
        ends = _spread(case, case["lo"], case["hi"], B)
        return [e - case["seq"] for e in ends], [case["seq"]] * B
    if case["op"] == "decode":
        return _spread(case, case["lo"], case["hi"], B), [0] * B
    if case["op"] == "step":
        return [e - 1 for e in _spread(case, case["lo"], case["hi"], B)], [1] * B
    starts = _spread(case, case["lo"], case["hi"], B)
    if case["hi"] == 0:  # fresh prompts of one length
        return starts, [case["seq"]] * B
    return starts, _spread(case, 1, case["seq"], B, salt=1)


def work(case):
    hq, hkv, D = case["hq"], case["hkv"], HEAD_DIM
    before, new = _plan(case)
    row = (hq + 2 * hkv) * D * 2  # a q|k|v row
    cached = 2 * hkv * ROW_BYTES  # a position's K and V in the cache
    tokens = sum(new)
    if case["op"] == "append":
        # q|k|v in; rotated q, the cache rows and their values out
        return {"bytes": tokens * (row + hq * D * 2 + cached + 2 * hkv * D * 2), "flops": tokens * 6 * (hq + hkv) * D}
    if case["op"] == "decode":
        T = sum(before)
        return {"bytes": T * cached + 2 * case["batch"] * hq * D * 2, "flops": 4 * T * hq * D}
    if case["op"] == "step":
        T = sum(before) + tokens
        return {"bytes": sum(before) * cached + tokens * (row + cached + hq * D * 2), "flops": 4 * T * hq * D}
    pairs = sum(n * s + n * (n + 1) // 2 for s, n in zip(before, new))
    T = sum(s + n for s, n in zip(before, new))
    return {"bytes": T * cached + 2 * tokens * hq * D * 2, "flops": 4 * pairs * hq * D}


# -- the cache's number format ---------------------------------------------------
def _quantise(x):
    """fp16 rows [..., 128] as codes in [-7, 7] and fp16 scales [..., 4]: the scale
    is the smallest number of 8 significant bits (and multiple of 2^-24) that is
    >= max|x| / 7, so that code * scale is exact in fp16; a zero group has scale
    1, and a row that is not finite has NaN scales."""
    g = x.double().reshape(*x.shape[:-1], HEAD_DIM // GROUP, GROUP)
    bad = ~torch.isfinite(g).all(dim=-1).all(dim=-1)
    g = torch.where(bad[..., None, None], torch.zeros((), dtype=g.dtype, device=g.device), g)
    top = g.abs().amax(dim=-1)
    m, e = torch.frexp(top / 7.0)
    s = torch.ldexp(torch.ceil(m * 256.0), e - 8)
    s = torch.where(s < 2.0 ** -16, torch.ceil(s * 2.0 ** 24) * 2.0 ** -24, s).clamp(max=9344.0)
    s = torch.where(top == 0, torch.ones_like(s), s)
    code = torch.round(g / s[..., None]).clamp(-7, 7).reshape(x.shape)
    s = torch.where(bad[..., None], torch.full_like(s, float("nan")), s)
    return code, s.half()


def _pack(code):
    n = (code + 8).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _parts(pool, page):
    """The code rows [..., page, 64] and scale rows [..., page, 4] of pool blocks."""
    return (pool[..., :page * 64].unflatten(-1, (page, 64)),
            pool[..., page * 64:].view(torch.float16).unflatten(-1, (page, 4)))


def _values(codes, scales, dtype):
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).to(dtype) - 8.0
    return (c.unflatten(-1, (HEAD_DIM // GROUP, GROUP)) * scales.to(dtype)[..., None]).flatten(-2)


# -- inputs ------------------------------------------------------------------------
def _pool(gen, n_pages, hkv, page, gain, dev):
    """Blocks of quantised rows; ``gain`` per (head, element) as the channels of real keys differ."""
    pool = torch.empty(n_pages, hkv, page * ROW_BYTES, dtype=torch.uint8, device=dev)
    codes, scales = _parts(pool, page)
    for a in range(0, n_pages, 2048):
        b = min(n_pages, a + 2048)
        x = (torch.randn(b - a, hkv, page, HEAD_DIM, generator=gen, device=dev) * gain[None, :, None]).half()
        c, s = _quantise(x)
        codes[a:b] = _pack(c)
        scales[a:b] = s
    return pool


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    B, hq, hkv, page, D = case["batch"], case["hq"], case["hkv"], case["page"], HEAD_DIM
    before, new = _plan(case)
    ends = [s + n for s, n in zip(before, new)]
    pages = -(-max(max(ends), 1) // page)
    n_pages = B * pages
    perm = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    i32 = dict(dtype=torch.int32, device=dev)
    s = dict(case=dict(case), max_seq_len=pages * page, page=page, ws=None)
    s["block_table"] = perm.view(B, pages).contiguous()
    gain = 1.0 + 3.0 * (torch.rand(hkv, D, generator=gen, device=dev) < 0.06).float()
    s["k_pool"] = _pool(gen, n_pages, hkv, page, gain, dev)
    s["v_pool"] = _pool(gen, n_pages, hkv, page, torch.ones_like(gain), dev)
    s["inv_freq"] = (1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)).float()
    q_dim, op = hq * D, case["op"]
    if op in ("append", "step"):
        rows = sum(new)
        qkv = torch.randn(rows, (hq + 2 * hkv) * D, generator=gen, device=dev)
        qkv[:, q_dim:q_dim + hkv * D] *= gain.reshape(1, -1)
        s["qkv"] = qkv.half()
        # a row of positions and of pages for each token, as the framework's append takes them
        start = torch.tensor(before, **i32)
        if op == "append" and case["seq"] > 1:
            s["pos"] = torch.arange(case["seq"], **i32).repeat(B) + start.repeat_interleave(case["seq"])
            s["rows_bt"] = s["block_table"].repeat_interleave(case["seq"], dim=0).contiguous()
        else:
            s["pos"], s["rows_bt"] = start, s["block_table"]
        if op == "append":
            s["q_out"] = torch.zeros(rows, q_dim, dtype=torch.float16, device=dev)
            s["k_out"] = torch.zeros(rows, hkv * D, dtype=torch.float16, device=dev)
            s["v_out"] = torch.zeros(rows, hkv * D, dtype=torch.float16, device=dev)
    if op in ("decode", "step"):
        s["seq_lens"] = torch.tensor(ends, **i32)
        s["out"] = torch.zeros(B, q_dim, dtype=torch.float16, device=dev)
    if op == "decode":
        s["q"] = torch.randn(B, q_dim, generator=gen, device=dev).half()
    if op == "prefill":
        s["q"] = torch.randn(B * case["seq"], q_dim, generator=gen, device=dev).half()
        s["out"] = torch.zeros(B * case["seq"], q_dim, dtype=torch.float16, device=dev)
        s["starts"], s["q_lens"] = torch.tensor(before, **i32), torch.tensor(new, **i32)
    s["error"] = torch.zeros(1, **i32)
    return s


# -- the plain forms -----------------------------------------------------------------
def _rotate(x, pos, inv_freq, style):
    """x [rows, heads, 128] rotated in 64 bits, rounded to fp16."""
    ang = pos.double()[:, None, None] * inv_freq.double()
    c, n = torch.cos(ang), torch.sin(ang)
    x = x.double()
    if style == 0:  # pairs (2j, 2j + 1)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * n, a * n + b * c], dim=-1).flatten(-2).half()
    a, b = x[..., :HEAD_DIM // 2], x[..., HEAD_DIM // 2:]  # pairs (j, j + 64)
    return torch.cat([a * c - b * n, a * n + b * c], dim=-1).half()


def _append(s):
    """Rotated q rows, and the K and V rows as the cache now holds them."""
    c, page = s["case"], s["page"]
    hq, hkv = c["hq"], c["hkv"]
    x = s["qkv"].unflatten(-1, (hq + 2 * hkv, HEAD_DIM))
    rot = _rotate(x[:, :hq + hkv], s["pos"], s["inv_freq"], c["style"])
    pos = s["pos"].long()
    pages = s["rows_bt"].gather(1, (pos // page)[:, None])[:, 0].long()
    kc, ks = _quantise(rot[:, hq:])
    vc, vs = _quantise(x[:, hq + hkv:])
    k_codes, k_scales = _parts(s["k_pool"], page)
    v_codes, v_scales = _parts(s["v_pool"], page)
    at = (pages, slice(None), pos % page)
    k_codes[at], k_scales[at] = _pack(kc), ks
    v_codes[at], v_scales[at] = _pack(vc), vs
    spread = lambda sc: sc.float().repeat_interleave(GROUP, dim=-1)  # noqa: E731
    k = (kc.float() * spread(ks)).half().flatten(1)
    v = (vc.float() * spread(vs)).half().flatten(1)
    return rot[:, :hq].flatten(1), k, v


def _gather(s, pool):
    """The cached rows of every sequence, fp32 [B, T, n_kv_heads, 128]."""
    page = s["page"]
    codes, scales = _parts(pool, page)
    bt = s["block_table"].long()
    x = _values(codes[bt], scales[bt], torch.float32)  # [B, pages, heads, page, 128]
    return x.transpose(2, 3).flatten(1, 2)


def _attend(s, q, lens):
    """q fp16 [B, S, heads, 128]; lens [B, S]: query (b, i) attends to the first lens[b, i] positions."""
    hkv = s["case"]["hkv"]
    B, S, hq, D = q.shape
    k, v = _gather(s, s["k_pool"]), _gather(s, s["v_pool"])
    g = q.float().view(B, S, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, D)  # [B, kv, G * S, D]
    scores = torch.matmul(g, k.permute(0, 2, 3, 1)).view(B, hkv, hq // hkv, S, -1).mul_(SCALE)
    mask = torch.arange(k.shape[1], device=q.device) >= lens[..., None]  # [B, S, T]
    scores.masked_fill_(mask[:, None, None], -float("inf"))
    scores -= scores.amax(dim=-1, keepdim=True)
    scores.exp_()
    total = scores.sum(dim=-1)
    o = torch.matmul(scores.view(B, hkv, -1, k.shape[1]), v.permute(0, 2, 1, 3)).view(B, hkv, hq // hkv, S, D)
    return (o / total[..., None]).permute(0, 3, 1, 2, 4).reshape(B, S, hq * D)


def _plain(s):
    c = s["case"]
    B, hq, hkv = c["batch"], c["hq"], c["hkv"]
    if c["op"] == "append":
        q, k, v = _append(s)
        s["q_out"].copy_(q)
        s["k_out"].copy_(k)
        s["v_out"].copy_(v)
        return s["q_out"], s["k_out"], s["v_out"], s["k_pool"], s["v_pool"]
    if c["op"] == "decode":
        o = _attend(s, s["q"].view(B, 1, hq, HEAD_DIM), s["seq_lens"][:, None])
        s["out"].copy_(o[:, 0])
        return s["out"]
    if c["op"] == "step":
        q, _, _ = _append(s)
        o = _attend(s, q.view(B, 1, hq, HEAD_DIM), s["seq_lens"][:, None])
        s["out"].copy_(o[:, 0])
        return s["out"], s["k_pool"], s["v_pool"]
    i = torch.arange(c["seq"], device=s["q"].device)
    o = _attend(s, s["q"].view(B, c["seq"], hq, HEAD_DIM), s["starts"][:, None] + i + 1)
    live = (i < s["q_lens"][:, None]).reshape(-1, 1)
    s["out"].copy_(torch.where(live, o.flatten(0, 1).half(), s["out"]))
    return s["out"]


# -- the framework's calls -------------------------------------------------------------
def _framework(s):
    from llamamps_b200 import kernels as K

    c = s["case"]
    hq, hkv, D, page = c["hq"], c["hkv"], HEAD_DIM, s["page"]
    if c["op"] == "append":
        K.rope_kv_append_q4(s["qkv"], s["pos"], s["inv_freq"], s["q_out"], s["k_pool"], s["v_pool"], s["rows_bt"],
                            page, hq, hkv, D, c["style"], k_out=s["k_out"], v_out=s["v_out"], error=s["error"])
        return s["q_out"], s["k_out"], s["v_out"], s["k_pool"], s["v_pool"]
    if c["op"] in ("decode", "step"):
        if s["ws"] is None:  # kept by a program from step to step
            s["splits"] = K.attention_q4_splits(c["batch"], hkv, s["max_seq_len"])
            size = K.attention_q4_workspace_size(c["batch"], hq, D, s["splits"])
            s["ws"] = torch.empty(max(size, 16), dtype=torch.uint8, device=s["out"].device)
        if c["op"] == "decode":
            return K.gqa_decode_attention_q4(s["q"], s["k_pool"], s["v_pool"], s["block_table"], s["seq_lens"],
                                             s["out"], s["ws"], page, hq, hkv, D, s["max_seq_len"], s["splits"],
                                             error=s["error"])
        K.gqa_decode_attention_rope_q4(s["qkv"], s["pos"], s["inv_freq"], s["k_pool"], s["v_pool"], s["block_table"],
                                       s["seq_lens"], s["out"], s["ws"], page, hq, hkv, D, s["max_seq_len"],
                                       s["splits"], c["style"], error=s["error"])
        return s["out"], s["k_pool"], s["v_pool"]
    if s["ws"] is None:
        s["splits"] = K.prefill_q4_splits(c["batch"], c["seq"], hq, hkv, s["max_seq_len"])
        size = K.prefill_q4_workspace_size(c["batch"], c["seq"], hq, D, s["splits"])
        s["ws"] = torch.empty(max(size, 16), dtype=torch.uint8, device=s["out"].device)
    return K.prefill_attention_q4(s["q"], s["k_pool"], s["v_pool"], s["block_table"], s["out"], c["batch"], c["seq"],
                                  page, hq, hkv, D, s["max_seq_len"], starts=s["starts"], q_lens=s["q_lens"],
                                  workspace=s["ws"], n_splits=s["splits"], error=s["error"])


def run(state):
    return _framework(state) if own else _plain(state)


# -- 64 bits -----------------------------------------------------------------------------
def _exact_rows(x):
    """Cached values of fp16 rows [rows, heads, 128], from the definition, in 64 bits."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for g in range(HEAD_DIM // GROUP):
        part = x[..., g * GROUP:(g + 1) * GROUP].double()
        need = part.abs().max(dim=-1, keepdim=True).values / 7.0
        # the grid of 8 significant bits around `need`: spacing 2^(floor(log2 need) - 7), never below 2^-24
        exp = torch.floor(torch.log2(need.clamp(min=2.0 ** -40)))
        step = torch.exp2(torch.clamp(exp - 7.0, min=-24.0))
        scale = torch.minimum(torch.ceil(need / step) * step, torch.full_like(need, 9344.0))
        scale[need == 0] = 1.0
        out[..., g * GROUP:(g + 1) * GROUP] = (part / scale).round().clamp(-7.0, 7.0) * scale
    return out


def _exact_turn(x, pos, inv_freq, style):
    """RoPE of [rows, heads, 128] by the 2 x 2 rotations, in 64 bits."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for j in range(HEAD_DIM // 2):
        i1, i2 = (2 * j, 2 * j + 1) if style == 0 else (j, j + HEAD_DIM // 2)
        t = (pos.double() * float(inv_freq[j]))[:, None]
        out[..., i1] = x[..., i1].double() * t.cos() - x[..., i2].double() * t.sin()
        out[..., i2] = x[..., i1].double() * t.sin() + x[..., i2].double() * t.cos()
    return out


def _exact_sequence(s, pool, b, n):
    """Rows 0 .. n-1 of sequence b, 64 bits [n, heads, 128]."""
    page, hkv = s["page"], s["case"]["hkv"]
    blocks = pool[s["block_table"][b, :-(-n // page)].long()]
    out = torch.empty(blocks.shape[0], page, hkv, HEAD_DIM, dtype=torch.float64, device=pool.device)
    bytes_ = blocks[:, :, :page * 64].reshape(-1, hkv, page, 64).permute(0, 2, 1, 3).int()
    scales = blocks[:, :, page * 64:].contiguous().view(torch.float16).reshape(-1, hkv, page, 4).permute(0, 2, 1, 3)
    out[..., 0::2] = (bytes_ % 16 - 8).double()
    out[..., 1::2] = (torch.div(bytes_, 16, rounding_mode="floor") - 8).double()
    for g in range(4):
        out[..., g * GROUP:(g + 1) * GROUP] *= scales[..., g:g + 1].double()
    return out.reshape(-1, hkv, HEAD_DIM)[:n]


def _exact_attention(q, k, v, first):
    """q [n, heads, 128]; query i attends to the first `first` + i positions."""
    n, hq, _ = q.shape
    out = torch.empty(n, hq, HEAD_DIM, dtype=torch.float64, device=q.device)
    seen = torch.arange(k.shape[0], device=q.device)[None] < first + torch.arange(n, device=q.device)[:, None]
    for h in range(hq):
        kv = h // (hq // k.shape[1])
        z = torch.where(seen, q[:, h].double() @ k[:, kv].T * SCALE, -math.inf)
        out[:, h] = torch.softmax(z, dim=-1) @ v[:, kv]
    return out.reshape(n, -1)


def exact(case, seed):
    s = prepare(case, seed)
    B, hq, hkv, D, op = case["batch"], case["hq"], case["hkv"], HEAD_DIM, case["op"]
    before, new = _plan(case)
    if op in ("append", "step"):
        x = s["qkv"].view(-1, hq + 2 * hkv, D)
        q = _exact_turn(x[:, :hq], s["pos"], s["inv_freq"], case["style"])
        # what the cache holds is a function of the rotated row rounded to fp16
        k_new = _exact_rows(_exact_turn(x[:, hq:hq + hkv], s["pos"], s["inv_freq"], case["style"]).half())
        v_new = _exact_rows(x[:, hq + hkv:])
        if op == "append":
            return q.flatten(1), k_new.flatten(1), v_new.flatten(1), None, None
    if op == "prefill":
        out = torch.zeros(B, case["seq"], hq * D, dtype=torch.float64, device=s["q"].device)
        q = s["q"].view(B, case["seq"], hq, D)
    else:
        out = torch.zeros(B, hq * D, dtype=torch.float64, device=s["out"].device)
        q = q.half() if op == "step" else s["q"].view(B, hq, D)
    for b in range(B):
        T = before[b] + new[b]
        k, v = _exact_sequence(s, s["k_pool"], b, T), _exact_sequence(s, s["v_pool"], b, T)
        if op == "prefill":
            out[b, :new[b]] = _exact_attention(q[b, :new[b]], k, v, before[b] + 1)
        else:
            if op == "step":
                k[-1], v[-1] = k_new[b], v_new[b]
            out[b] = _exact_attention(q[b][None], k, v, T)[0]
    if op == "prefill":
        return out.flatten(0, 1)
    return out if op == "decode" else (out, None, None)
