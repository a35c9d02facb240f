"""The 4-bit K/V cache and the attention over it, as cases to time and to compare.

The pool.  Sixteen slots are a block; a pool is ``(num_blocks, num_kv_heads, 9 * head_dim / 2)``
elements of the 16-bit type: per block and head the codes of sixteen rows (``head_dim / 2`` bytes
each), then sixteen rows of (scale, bias) pairs, one pair for every 64 elements of a row.  A group of 64 elements
is held as ``scale * code + bias`` with

    bias = min,  scale = round16((max - min) / 15),  code = min(15, rint((x - bias) / scale))

(a scale below 2^-100 is 0, and then every code is).  Word ``r * (head_dim / 64) + g`` (32 bits) of a row holds elements
``64 g + 8 r`` .. ``64 g + 8 r + 7``, element ``e`` of them in nibble ``e / 2 + 4 (e % 2)``.

Kinds of cases: ``store`` (append rows, and read the pool back), ``project`` (norm, rotation and append in one, and read the pool
back), ``decode`` and ``prefill`` (attention).  A pool's values come back through the pool's own reading operator.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 64
BLOCK = 16

# No drawn case costs more than the largest listed ones (bytes that must move, operations).
MAX_BYTES = 7.0e8
MAX_FLOPS = 1.3e12


def _case(name=None, *, kind, hq=32, hkv=8, head_dim=128, dtype="bf16", page_size=16, batch=1, lens=1, kv_lo=0, kv_hi=0,
          q_lo=1, q_hi=1, rotary=0, norm=True, gate=False, window=0, cross=False):
    """``kv_lo`` .. ``kv_hi``: cached tokens of a request in front of its ``q_lo`` .. ``q_hi`` new ones (decode: its length).
    ``store`` and ``project`` have ``q_lo`` rows for each of ``batch`` requests.  ``rotary`` 0: the whole head."""
    c = dict(kind=kind, hq=hq, hkv=hkv, head_dim=head_dim, dtype=dtype, page_size=page_size, batch=batch, lens=lens,
             kv_lo=kv_lo, kv_hi=kv_hi, q_lo=q_lo, q_hi=q_hi, rotary=rotary, norm=norm, gate=gate, window=window, cross=cross)
    return c if name is None else dict(name=name, **c)


def listed():
    return [
        # A decode step of a small batch puts one row per request into the pool: all latency.
        _case("append_decode_rows", kind="store", batch=24, hq=16),
        # Prompts put into the pool by layers that rotate their own keys, 256-wide heads, f16.
        _case("append_prompts_d256_f16", kind="store", hq=16, hkv=2, head_dim=256, dtype="f16", batch=3, q_lo=1777),
        # A long prompt's rows: the largest append, all traffic.
        _case("append_long_prompt", kind="store", batch=2, q_lo=24576),
        # A decode step of a layer with q/k norms.
        _case("project_decode_rows", kind="project", batch=61),
        # A prefill step of gated 256-wide layers that rotate a quarter of the head, far into a document.
        _case("project_prompts_d256", kind="project", hq=16, hkv=4, head_dim=256, rotary=64, batch=2, q_lo=3000, kv_lo=90000),
        # One user chatting with a small model: the smallest attention call, all latency.
        _case("decode_one_request", kind="decode", hq=16, kv_lo=700, kv_hi=700),
        # Gated layers with 256-wide heads, ragged, f16.
        _case("decode_gated_d256_f16", kind="decode", hq=16, hkv=2, head_dim=256, dtype="f16", gate=True, batch=19, lens=11,
              kv_lo=512, kv_hi=16384),
        # Long-context continuous batching: the largest decode, all K/V traffic.
        _case("decode_long_context", kind="decode", batch=32, lens=505, kv_lo=4096, kv_hi=32768),
        # Speculative verification: five tokens a request over contexts of very different lengths.
        _case("verify_five_tokens", kind="prefill", hkv=4, page_size=32, batch=16, lens=404, kv_lo=1024, kv_hi=16384, q_lo=5,
              q_hi=5),
        # A draft layer's blocks under a sliding window.
        _case("draft_window_block", kind="prefill", batch=16, lens=303, kv_lo=6000, kv_hi=8176, q_lo=16, q_hi=16, window=4096,
              cross=True),
        # Chunked prefill over cached prefixes: the ordinary prefill step.
        _case("prefill_chunked", kind="prefill", batch=4, lens=202, kv_lo=1000, kv_hi=4096, q_lo=300, q_hi=512),
        # A chunk of a long document: the largest prefill, all tensor-core work.
        _case("prefill_long_document", kind="prefill", kv_lo=16384, kv_hi=16384, q_lo=4096, q_hi=4096),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Rows of one to some ten thousand tokens; decode of 1 to 64 requests; prefill of 2 to 4096 new tokens a request, with and
    without windows; both head sizes and types, the head layouts of the listed cases and those between."""
    while True:
        kind = rng.choice(("store", "project", "decode", "decode", "prefill", "prefill"))
        wide = rng.random() < 0.35
        hq, hkv = rng.choice(((16, 2), (16, 4), (24, 4), (32, 2)) if wide else ((16, 8), (32, 8), (32, 4), (40, 8), (8, 8)))
        c = dict(kind=kind, hq=hq, hkv=hkv, head_dim=256 if wide else 128, dtype=rng.choice(("bf16", "bf16", "f16")),
                 page_size=rng.choice((16, 16, 16, 32, 64)), lens=rng.randrange(1, 1 << 20))
        if kind in ("store", "project"):
            c.update(batch=_log(rng, 1, 48), q_lo=rng.choice((1, _log(rng, 2, 8192))), kv_lo=_log(rng, 1, 100000),
                     rotary=rng.choice((0, 64, 128)) if wide else rng.choice((0, 0, 64)), norm=rng.random() < 0.8)
        elif kind == "decode":
            lo = _log(rng, 1, 16384)
            c.update(batch=_log(rng, 1, 64), kv_lo=lo, kv_hi=_log(rng, lo, 32768), gate=rng.random() < 0.3)
        else:
            q_lo = _log(rng, 2, 2048)
            lo = rng.choice((0, _log(rng, 64, 12000)))
            c.update(batch=_log(rng, 1, 24), kv_lo=lo, kv_hi=max(lo, rng.choice((0, _log(rng, 64, 16384)))), q_lo=q_lo,
                     q_hi=_log(rng, q_lo, 4096), window=rng.choice((0, 0, _log(rng, 64, 4096))), cross=rng.random() < 0.2,
                     gate=rng.random() < 0.2)
        case = _case(**c)
        w = work(case)
        total = sum(q * (p + q) for p, q in _lengths(case)) * hq if kind == "prefill" else 0
        padded = case["batch"] * max(p + q for p, q in _lengths(case)) * hkv * case["head_dim"]
        if w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS and total <= 3e9 and padded <= 1.2e9:
            return case


def _lengths(case):
    """(cached, new) tokens of every request, the same for every seed."""
    import random

    rng = random.Random(case["lens"])
    if case["kind"] in ("store", "project"):
        return [(case["kv_lo"] + 37 * i, case["q_lo"]) for i in range(case["batch"])]
    out = []
    for i in range(case["batch"]):
        kv = case["kv_hi"] if i == 0 else int(round(math.exp(rng.uniform(math.log(max(1, case["kv_lo"])),
                                                                         math.log(max(1, case["kv_hi"]))))))
        if case["kv_hi"] == 0:
            kv = 0
        q = rng.randint(case["q_lo"], case["q_hi"])
        out.append((max(0, kv - 1), 1) if case["kind"] == "decode" else (kv, q))
    return out


def work(case):
    d, hq, hkv = case["head_dim"], case["hq"], case["hkv"]
    row4 = hkv * (d // 2 + d // 16)            # bytes of a token's codes, scales and biases, of K or V
    lens = _lengths(case)
    n = sum(q for _, q in lens)
    if case["kind"] in ("store", "project"):
        slots = _slots(case)
        back = 2 * slots * (row4 + hkv * d * 2)
        q_io = 2 * n * hq * d * 2 if case["kind"] == "project" else 0
        return {"bytes": 2 * n * (hkv * d * 2 + row4) + q_io + back, "flops": 0}
    pairs = keys = 0
    for p, q in lens:
        w = case["window"]
        for t in range(q) if case["kind"] == "prefill" else (0,):
            hi = p + q if case["cross"] else p + t + 1
            pairs += hi - (max(0, p + t - w + 1) if w else 0)
        keys += p + q - (max(0, p - w + 1) if w else 0)
    return {"bytes": 2 * keys * row4 + n * hq * d * 2 * (3 if case["gate"] else 2), "flops": 4 * d * hq * pairs}


def _slots(case):
    """Slots of the pool of a case."""
    ps = case["page_size"]
    pages = sum(-(-(q if case["kind"] in ("store", "project") else p + q) // ps) for p, q in _lengths(case))
    return (pages + max(2, pages // 16)) * ps


# ------------------------------------------------------------------ the plain form of the pool
def _quantise(x):
    """(codes, scale, bias) of rows (..., head_dim) of a 16-bit type: codes as numbers, scale and bias in that type."""
    g = x.double().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / 15).float().to(x.dtype)
    scale = torch.where(scale.double() < 2.0 ** -100, torch.zeros_like(scale), scale)
    s = scale.double().unsqueeze(-1)
    code = torch.where(s > 0, ((g - lo.unsqueeze(-1)) / torch.where(s > 0, s, torch.ones_like(s))).round(), torch.zeros_like(g))
    return code.clamp(0, 15).to(torch.int32), scale, lo.to(x.dtype)


def _row_parts(pool, head_dim):
    """Views of a pool: code words (blocks, heads, 16, words) int32 and pairs (blocks, heads, 16, groups, 2)."""
    codes = BLOCK * head_dim // 4
    words = pool[..., :codes].view(torch.int32).unflatten(-1, (BLOCK, head_dim // 8))
    pairs = pool[..., codes:].unflatten(-1, (BLOCK, head_dim // GROUP, 2))
    return words, pairs


def _nibble_shift(device):
    e = torch.arange(8, device=device)
    return 4 * (e // 2 + 4 * (e % 2))


def _pack(code):
    """(..., groups, 64) codes -> (..., words) int32."""
    w = code.unflatten(-1, (8, 8)).long() << _nibble_shift(code.device)
    w = w.sum(-1).transpose(-1, -2).flatten(-2)            # word r * groups + g
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _append(pool, rows, slots, head_dim):
    code, scale, bias = _quantise(rows)
    words, pairs = _row_parts(pool, head_dim)
    s = slots.long()
    words[s // BLOCK, :, s % BLOCK] = _pack(code)
    pairs[s // BLOCK, :, s % BLOCK] = torch.stack((scale, bias), -1)


def _values(words, pairs):
    """float32 values (..., head_dim) of code words (..., words) and their pairs (..., groups, 2)."""
    groups = pairs.shape[-2]
    w = words.unflatten(-1, (8, groups)).transpose(-1, -2).unsqueeze(-1)          # (..., groups, 8, 1)
    code = (w >> _nibble_shift(words.device).int()) & 15
    scale, bias = pairs[..., 0].float(), pairs[..., 1].float()
    return (code.flatten(-2).float() * scale.unsqueeze(-1) + bias.unsqueeze(-1)).flatten(-2)


def _read(pool, slots, head_dim):
    words, pairs = _row_parts(pool, head_dim)
    s = slots.long()
    return _values(words[s // BLOCK, :, s % BLOCK], pairs[s // BLOCK, :, s % BLOCK])


# ------------------------------------------------------------------ inputs
def _rows(gen, dtype, n, heads, d):
    """Keys or values as projections give them: normal, some channels much larger, a few rows offset."""
    dev = "cuda"
    channel = 0.5 + 1.5 * torch.rand(heads, d, generator=gen, device=dev)
    channel = channel * torch.where(torch.rand(heads, d, generator=gen, device=dev) < 0.03, 6.0, 1.0)
    shift = 0.5 * torch.randn(heads, d, generator=gen, device=dev)
    return (torch.randn(n, heads, d, generator=gen, device=dev) * channel + shift).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dev, T, d = "cuda", DTYPES[case["dtype"]], case["head_dim"]
    hq, hkv, ps = case["hq"], case["hkv"], case["page_size"]
    lens = _lengths(case)
    n, slots = sum(q for _, q in lens), _slots(case)
    s = dict(case=case, slots=slots)
    held = [q if case["kind"] in ("store", "project") else p + q for p, q in lens]
    pages = [-(-t // ps) for t in held]
    order = torch.randperm(slots // ps, generator=gen, device=dev)[:sum(pages)].int()
    shape = (slots // BLOCK, hkv, 9 * d // 2)
    s["k_cache"] = torch.zeros(shape, dtype=T, device=dev)
    s["v_cache"] = torch.zeros(shape, dtype=T, device=dev)
    if case["kind"] in ("store", "project"):
        starts = torch.tensor([0] + pages[:-1]).cumsum(0)
        at = torch.cat([torch.arange(t) + int(a) * ps for t, a in zip(held, starts)]).to(dev)
        s["out_loc"] = (order[at // ps] * ps + at % ps).int()
        # (one projection's output, cut into its heads: rows with a stride)
        qkv = _rows(gen, T, n, (hq if case["kind"] == "project" else 0) + 2 * hkv, d)
        s["q"], s["k"], s["v"] = qkv.split((qkv.shape[1] - 2 * hkv, hkv, hkv), 1)
        s["all_slots"] = torch.arange(slots, dtype=torch.int32, device=dev)
        if case["kind"] == "project":
            s["positions"] = torch.cat([torch.arange(p, p + q) for p, q in lens]).int().to(dev)
            for w in ("q_weight", "k_weight"):
                s[w] = (1 + 0.2 * torch.randn(d, generator=gen, device=dev)).to(T) if case["norm"] else None
        return s
    # a pool that the requests (and others before them) have filled
    step = max(16, (1 << 26) // (hkv * d) // 16 * 16)
    for a in range(0, slots, step):
        m = min(step, slots - a)
        at = torch.arange(a, a + m, device=dev)
        for name in ("k_cache", "v_cache"):
            _append(s[name], _rows(gen, T, m, hkv, d), at, d)
    s["q"] = torch.randn(n, hq, d, generator=gen, device=dev).to(T)
    s["gate"] = torch.randn(n, hq, d, generator=gen, device=dev).to(T) if case["gate"] else None

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s["page_indptr"] = ints([0] + torch.tensor(pages).cumsum(0).tolist())
    s["page_indices"] = order
    s["kv_lens"] = ints(held)
    s["scale"] = 1 / math.sqrt(d)
    if case["kind"] == "prefill":
        new = [q for _, q in lens]
        s["qo_indptr"] = ints([0] + torch.tensor(new).cumsum(0).tolist())
        s["prefix_lens"] = ints([p for p, _ in lens])
        s["max_new"] = max(new)
    s["max_kv"] = max(held)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"store": _own_store, "project": _own_project, "decode": _own_decode, "prefill": _own_prefill}[kind](s)
    return {"store": _store, "project": _project, "decode": _decode, "prefill": _prefill}[kind](s)


def _own_store(s):
    from mini_sglang_mlx_b200 import kernel as K

    K.store_kv_cache_q4(s["k_cache"], s["v_cache"], s["out_loc"], s["k"], s["v"])
    return K.load_kv_cache_q4(s["k_cache"], s["v_cache"], s["all_slots"])


def _own_project(s):
    from mini_sglang_mlx_b200 import kernel as K

    c = s["case"]
    q = K.qk_norm_rope_store_q4(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["positions"], s["out_loc"],
                                s["k_cache"], s["v_cache"], rope_base=1e6, eps=1e-6, rotary_dim=c["rotary"] or c["head_dim"])
    return (q, *K.load_kv_cache_q4(s["k_cache"], s["v_cache"], s["all_slots"]))


def _own_decode(s):
    from mini_sglang_mlx_b200 import kernel as K

    return K.paged_decode_attention_q4(s["q"], s["k_cache"], s["v_cache"], s["page_indptr"], s["page_indices"], s["kv_lens"],
                                       s["scale"], page_size=s["case"]["page_size"], gate=s["gate"])


def _own_prefill(s):
    from mini_sglang_mlx_b200 import kernel as K

    c = s["case"]
    return K.paged_prefill_attention_q4(s["q"], s["k_cache"], s["v_cache"], s["qo_indptr"], s["page_indptr"],
                                        s["page_indices"], s["kv_lens"], s["prefix_lens"], s["scale"], s["max_new"],
                                        page_size=c["page_size"], is_cross_attention=c["cross"],
                                        sliding_window_size=c["window"], gate=s["gate"])


def _store(s):
    c = s["case"]
    d, T = c["head_dim"], DTYPES[c["dtype"]]
    _append(s["k_cache"], s["k"], s["out_loc"], d)
    _append(s["v_cache"], s["v"], s["out_loc"], d)
    return tuple(_read(s[name], s["all_slots"], d).to(T) for name in ("k_cache", "v_cache"))


def _norm_rotate(x, weight, positions, rotary, eps=1e-6, base=1e6):
    """RMSNorm (rounded to the type, as the layer's own norm gives it), then the rotation of the first ``rotary`` elements,
    pairs (i, i + rotary / 2)."""
    T, y = x.dtype, x.float()
    if weight is not None:
        y = (y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * weight.float()).to(T).float()
    half = rotary // 2
    freq = base ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    angle = positions.double()[:, None, None] * freq
    cos, sin = angle.cos().float(), angle.sin().float()
    a, b = y[..., :half], y[..., half:rotary]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, y[..., rotary:]), -1).to(T)


def _project(s):
    c = s["case"]
    d, T = c["head_dim"], DTYPES[c["dtype"]]
    rotary = c["rotary"] or d
    q = _norm_rotate(s["q"], s["q_weight"], s["positions"], rotary)
    _append(s["k_cache"], _norm_rotate(s["k"], s["k_weight"], s["positions"], rotary), s["out_loc"], d)
    _append(s["v_cache"], s["v"], s["out_loc"], d)
    return (q, *(_read(s[name], s["all_slots"], d).to(T) for name in ("k_cache", "v_cache")))


def _padded_slots(s):
    """(batch, longest) slot ids, and which of them are a request's."""
    ps = s["case"]["page_size"]
    t = torch.arange(s["max_kv"], device="cuda")
    first, last = s["page_indptr"][:-1].long(), s["page_indptr"][1:].long()
    page = torch.minimum(first[:, None] + t // ps, (last - 1)[:, None])
    return s["page_indices"][page].long() * ps + t % ps, t < s["kv_lens"][:, None]


def _attend(q, k, v, mask, scale):
    """q (batch, new, hkv, group, d); k, v (batch, keys, hkv, d); mask (batch, new, keys); rows without a key give zeros."""
    score = torch.einsum("bnhgd,bthd->bhgnt", q, k).mul_(scale)
    score.masked_fill_(~mask[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top.isfinite(), top, torch.zeros_like(top))).exp_()
    total = score.sum(-1, keepdim=True)
    score.div_(torch.where(total > 0, total, torch.ones_like(total)))
    return torch.einsum("bhgnt,bthd->bnhgd", score, v)


def _gated(out, gate, T):
    """The layer's gate is an operation of its own behind the attention: output and sigmoid are each of the 16-bit type."""
    out = out.to(T)
    return out if gate is None else (out.float() * torch.sigmoid(gate.float()).to(T).float()).to(T)


def _decode(s):
    c = s["case"]
    d, hkv = c["head_dim"], c["hkv"]
    at, mask = _padded_slots(s)
    k, v = _read(s["k_cache"], at, d), _read(s["v_cache"], at, d)
    q = s["q"].float().unflatten(1, (hkv, -1)).unsqueeze(1)
    out = _attend(q, k, v, mask[:, None], s["scale"])
    return _gated(out.reshape(s["q"].shape), s["gate"], s["q"].dtype)


def _prefill(s):
    c = s["case"]
    d, hkv = c["head_dim"], c["hkv"]
    at, held = _padded_slots(s)
    k, v = _read(s["k_cache"], at, d), _read(s["v_cache"], at, d)
    begin, end = s["qo_indptr"][:-1].long(), s["qo_indptr"][1:].long()
    i = torch.arange(s["max_new"], device="cuda")
    row = torch.minimum(begin[:, None] + i, (end - 1)[:, None])
    q = s["q"][row].float().unflatten(2, (hkv, -1))
    pos = (s["prefix_lens"].long()[:, None] + i)[..., None]
    t = torch.arange(s["max_kv"], device="cuda")
    mask = held[:, None] & ((t <= pos) if not c["cross"] else torch.ones_like(t <= pos))
    if c["window"]:
        mask = mask & (t > pos - c["window"])
    out = _attend(q, k, v, mask, s["scale"]).flatten(2, 3)
    real = i < (end - begin)[:, None]
    return _gated(out[real], s["gate"], s["q"].dtype)


# ------------------------------------------------------------------ 64 bits
def _exact_codes(x):
    """Values (n, heads, d) in float64 that rows of a 16-bit type stand for once they are held in the pool."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for g in range(x.shape[-1] // GROUP):
        part = x[..., g * GROUP:(g + 1) * GROUP].double()
        lo = part.min(-1, keepdim=True).values
        scale = ((part.max(-1, keepdim=True).values - lo) / 15).to(x.dtype).double()
        n = torch.where(scale >= 2.0 ** -100, torch.clamp(torch.round((part - lo) / scale), max=15.0), 0.0)
        out[..., g * GROUP:(g + 1) * GROUP] = torch.where(n > 0, n * scale, 0.0) + lo
    return out


def _exact_pool(pool, slots, d):
    """float64 values (len(slots), heads, d), byte by byte."""
    raw = pool.view(torch.uint8)
    b, r = slots.long() // BLOCK, slots.long() % BLOCK
    codes = raw[..., :8 * d].reshape(*raw.shape[:2], BLOCK, d // 2)[b, :, r].long()        # (n, heads, bytes)
    pairs = raw[..., 8 * d:].contiguous().view(pool.dtype).reshape(*raw.shape[:2], BLOCK, -1, 2)[b, :, r].double()
    groups, out = d // GROUP, torch.empty(len(slots), pool.shape[1], d, dtype=torch.float64, device=pool.device)
    for i in range(d):
        g, rest = divmod(i, GROUP)
        r8, e = divmod(rest, 8)
        nibble = e // 2 + 4 * (e % 2)
        byte = codes[..., 4 * (r8 * groups + g) + nibble // 2]
        out[..., i] = pairs[..., g, 0] * ((byte >> (4 * (nibble % 2))) & 15) + pairs[..., g, 1]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    d, hq, hkv, T = case["head_dim"], case["hq"], case["hkv"], DTYPES[case["dtype"]]
    if case["kind"] in ("store", "project"):
        k, q = s["k"], None
        if case["kind"] == "project":
            rd = case["rotary"] or d
            turned = []
            for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
                y = x.double()
                if w is not None:
                    y = (y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + 1e-6) * w.double()).to(T).double()
                z = y.clone()
                for i in range(rd // 2):
                    a = s["positions"].double()[:, None] * 1e6 ** (-2 * i / rd)
                    z[..., i] = y[..., i] * a.cos() - y[..., i + rd // 2] * a.sin()
                    z[..., i + rd // 2] = y[..., i + rd // 2] * a.cos() + y[..., i] * a.sin()
                turned.append(z)
            q, k = turned[0], turned[1].to(T)
        out = []
        for x in (k, s["v"]):
            pool = torch.zeros(s["slots"], hkv, d, dtype=torch.float64, device="cuda")
            pool[s["out_loc"].long()] = _exact_codes(x)
            out.append(pool)
        return tuple(out) if q is None else (q, *out)
    ps, result = case["page_size"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    indptr, lens = s["page_indptr"].tolist(), s["kv_lens"].tolist()
    qo = s["qo_indptr"].tolist() if case["kind"] == "prefill" else list(range(len(lens) + 1))
    for b, length in enumerate(lens):
        t = torch.arange(length, device="cuda")
        slots = s["page_indices"][indptr[b]:indptr[b + 1]].long()[t // ps] * ps + t % ps
        k, v = _exact_pool(s["k_cache"], slots, d), _exact_pool(s["v_cache"], slots, d)
        new = qo[b + 1] - qo[b]
        pos = (length - new + torch.arange(new, device="cuda"))[:, None]
        seen = (t <= pos) | bool(case["cross"] or case["kind"] == "decode")
        if case["window"]:
            seen = seen & (t >= pos - case["window"] + 1)
        for h in range(hq):
            kv = h // (hq // hkv)
            score = (s["q"][qo[b]:qo[b + 1], h].double() @ k[:, kv].T) * s["scale"]
            p = torch.softmax(torch.where(seen, score, -math.inf), -1)
            result[qo[b]:qo[b + 1], h] = p @ v[:, kv]
    if s["gate"] is not None:
        result = result * torch.sigmoid(s["gate"].double())
    return result
