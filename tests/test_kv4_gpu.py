"""The 4-bit K/V pool: rows in and out, norm + rotation + append, decode and prefill, against 64-bit references."""
import math

import pytest
import torch

from mini_sglang_mlx_b200 import _lib
from mini_sglang_mlx_b200 import kernel as K
from oracle import kv4_oracle as Q
from oracle import paged_attention_oracle as O

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
LAYOUTS = [(BF16, 128), (F16, 128), (BF16, 256), (F16, 256)]


def half_unit(dtype):
    return torch.finfo(dtype).eps / 2


def pools(num_slots, hkv, d, dtype, fill=None):
    shape = K.kv_cache_q4_shape(num_slots, hkv, d)
    out = [torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2)]
    if fill is not None:
        for t in out:
            t.view(torch.uint8).fill_(fill)
    return out


def rows(gen, n, heads, d, dtype, spread=1.0):
    x = torch.randn(n, heads, d, generator=gen) * spread + 0.4 * torch.randn(heads, d, generator=gen)
    return x.to(dtype)


def clean():
    assert K.device_status() == 0


def same_bytes(a, b):
    assert torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


# ------------------------------------------------------------------ rows in
@pytest.mark.parametrize("dtype,d", LAYOUTS)
@pytest.mark.parametrize("n,hkv", [(1, 1), (3, 8), (77, 2), (300, 5)])
def test_store_writes_the_bytes_of_the_format(dtype, d, n, hkv):
    clean()
    gen = torch.Generator().manual_seed(n * hkv + d)
    num_slots = 16 * (n // 8 + 2)
    k, v = rows(gen, n, hkv, d, dtype), rows(gen, n, hkv, d, dtype, 30.0)
    slots = torch.randperm(num_slots, generator=gen)[:n].int()
    kc, vc = pools(num_slots, hkv, d, dtype, fill=0x5a)
    kr, vr = kc.cpu(), vc.cpu()
    Q.write(kr, k, slots)
    Q.write(vr, v, slots)
    K.store_kv_cache_q4(kc, vc, slots.cuda(), k.cuda(), v.cuda())
    same_bytes(kc, kr)          # (the other slots' bytes as they were)
    same_bytes(vc, vr)
    clean()


@pytest.mark.parametrize("dtype,d", LAYOUTS)
def test_store_of_hard_rows(dtype, d):
    """Halves between two codes, equal elements, subnormal and huge ranges, signed zeros, one outlier."""
    big = Q.LARGEST
    tiny = torch.finfo(dtype).smallest_normal
    gen = torch.Generator().manual_seed(5)
    x = torch.zeros(40, 2, d, dtype=torch.float64)
    x[0] = 3.25
    x[1] = torch.arange(d).remainder(31) * 0.5                       # scale 1: every second element is a half
    x[2] = torch.arange(d).remainder(16) * 77 / 256 * 0.5
    x[3, :, ::3] = big
    x[3, :, 1::3] = -big
    x[4] = torch.randn(2, d, generator=gen) * tiny
    x[5, :, 5] = 1e4
    x[6] = -0.0
    x[7, 0, :64] = torch.arange(64) * 2.0 ** -20
    x[8] = big
    x[9] = torch.arange(d) * tiny / 8
    for i in range(10, 40):                                          # short numbers: many ties
        x[i] = torch.randint(0, 200, (2, d), generator=gen).double() * 2.0 ** (i % 7 - 5)
    k = x.to(dtype)
    v = -x.flip(0).to(dtype)
    slots = torch.arange(40).int()
    kc, vc = pools(48, 2, d, dtype)
    kr, vr = kc.cpu(), vc.cpu()
    Q.write(kr, k, slots)
    Q.write(vr, v, slots)
    K.store_kv_cache_q4(kc, vc, slots.cuda(), k.cuda(), v.cuda())
    assert torch.equal(Q.read(kc, slots), Q.read(kr, slots))         # (values: the sign of a zero bias is open)
    assert torch.equal(Q.read(vc, slots), Q.read(vr, slots))
    clean()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_store_of_numbers_that_are_not_finite(dtype):
    gen = torch.Generator().manual_seed(1)
    k = rows(gen, 6, 2, 128, dtype)
    k[0, 0, 3] = math.inf
    k[1, 1, 70] = -math.inf
    k[2, 0, 9] = math.nan
    k[3] = math.nan
    k[4, 1, 100] = 40000.0
    k[4, 0, 1] = -65504.0
    v = k.flip(0).contiguous()
    kc, vc = pools(16, 2, 128, dtype)
    kr, vr = kc.cpu(), vc.cpu()
    slots = torch.tensor([4, 9, 0, 1, 15, 7]).int()
    Q.write(kr, k, slots)
    Q.write(vr, v, slots)
    K.store_kv_cache_q4(kc, vc, slots.cuda(), k.cuda(), v.cuda())
    assert torch.equal(Q.read(kc, slots), Q.read(kr, slots)) and torch.equal(Q.read(vc, slots), Q.read(vr, slots))
    assert K.device_status() & 4
    clean()


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 256)])
@pytest.mark.parametrize("pad", [0, 4, 8])
def test_store_of_views_and_padded_rows(dtype, d, pad):
    """Rows of a fused projection (any stride, 8-byte aligned), a padded batch, indices outside the pool, an empty call."""
    clean()
    gen = torch.Generator().manual_seed(2)
    n, hkv = 21, 4
    fused = rows(gen, n, 3 * hkv, d, dtype).view(n, -1)
    wide = torch.zeros(n, fused.shape[1] + pad, dtype=dtype)
    wide[:, pad:] = fused
    dev = wide.cuda()[:, pad:]
    k = dev[:, hkv * d:2 * hkv * d].unflatten(1, (hkv, d))
    v = dev[:, 2 * hkv * d:].unflatten(1, (hkv, d))
    slots = torch.randperm(64, generator=gen)[:n].int()
    slots[3], slots[8], slots[20] = -1, 64, 2 ** 31 - 1
    kc, vc = pools(64, hkv, d, dtype, fill=0x11)
    kr, vr = kc.cpu(), vc.cpu()
    Q.write(kr, k.cpu(), slots)
    Q.write(vr, v.cpu(), slots)
    K.store_kv_cache_q4(kc, vc, slots.cuda(), k, v)
    same_bytes(kc, kr)
    same_bytes(vc, vr)
    assert K.device_status() == 2
    K.store_kv_cache_q4(kc, vc, slots[:0].cuda(), k[:0], v[:0])
    same_bytes(kc, kr)


# ------------------------------------------------------------------ rows out
@pytest.mark.parametrize("dtype,d", LAYOUTS)
@pytest.mark.parametrize("n", [1, 50, 333])
def test_load_gives_the_rounded_values(dtype, d, n):
    clean()
    gen = torch.Generator().manual_seed(n)
    hkv = 3
    kc, vc = pools(352, hkv, d, dtype)
    every = torch.arange(352).int().cuda()
    K.store_kv_cache_q4(kc, vc, every, rows(gen, 352, hkv, d, dtype).cuda(), rows(gen, 352, hkv, d, dtype, 9.0).cuda())
    at = torch.randint(0, 352, (n,), generator=gen).int()            # (the same slot may be read twice)
    if n > 1:
        at[n // 2] = -3
        at[1] = 352
    got = K.load_kv_cache_q4(kc, vc, at.cuda())
    for x, pool in zip(got, (kc, vc)):
        ref = Q.read(pool, at)
        assert x.shape == (n, hkv, d) and x.dtype == dtype
        # one rounding of an fp32 fma: half a unit of the type and of fp32
        assert ((x.double().cpu() - ref).abs() <= (half_unit(dtype) + 2.0 ** -23) * ref.abs() + 1e-7).all()
    assert K.device_status() == (2 if n > 1 else 0)


# ------------------------------------------------------------------ norm, rotation, append
def norm_rotate(x, w, pos, rd, eps, base):
    """In 64 bits, the norm's result rounded to the type."""
    y = x.double()
    if w is not None:
        y = (y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()).to(x.dtype).double()
    h = rd // 2
    a = pos.double()[:, None] * base ** (-torch.arange(h, dtype=torch.float64) / h)
    c, s = a.cos()[:, None], a.sin()[:, None]
    return torch.cat((y[..., :h] * c - y[..., h:rd] * s, y[..., h:rd] * c + y[..., :h] * s, y[..., rd:]), -1), y


@pytest.mark.parametrize("dtype,d,rd", [(BF16, 128, 128), (F16, 128, 64), (BF16, 256, 64), (F16, 256, 256), (BF16, 256, 128),
                                        (F16, 128, 32)])
@pytest.mark.parametrize("n,hq,hkv,norm", [(1, 1, 1, True), (5, 16, 2, True), (130, 6, 3, False), (67, 9, 5, True)])
def test_project_and_store(dtype, d, rd, n, hq, hkv, norm):
    clean()
    gen = torch.Generator().manual_seed(n + rd)
    fused = rows(gen, n, hq + 2 * hkv, d, dtype)
    q, k, v = fused.cuda().split((hq, hkv, hkv), 1)
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=gen)).to(dtype) if norm else None for _ in range(2))
    pos = torch.randint(0, 200000, (n,), generator=gen).int()
    slots = torch.randperm(16 * (n // 16 + 2), generator=gen)[:n].int()
    if n > 5:
        slots[2] = -1
    kc, vc = pools(16 * (n // 16 + 2), hkv, d, dtype)
    before = q.clone()
    out = K.qk_norm_rope_store_q4(q, k, v, None if qw is None else qw.cuda(), None if kw is None else kw.cuda(), pos.cuda(),
                                  slots.cuda(), kc, vc, rope_base=1e6, eps=1e-6, rotary_dim=rd)
    assert torch.equal(q, before) and out.is_contiguous() and out.shape == (n, hq, d)
    u = half_unit(dtype)
    ref, normed = norm_rotate(q.cpu(), qw, pos, rd, 1e-6, 1e6)
    # the norm's rounding can fall the other way (a unit of either member of a pair), then one rounding; the angle's sine is off by
    # 2^-20 at most
    size = normed.abs() + torch.cat((normed[..., rd // 2:rd], normed[..., :rd // 2], 0 * normed[..., rd:]), -1).abs()
    tol = (3 * u + 2.0 ** -19) * size + 1e-7
    assert ((out.double().cpu() - ref).abs() <= tol).all()
    # almost all of them do not: a rounding flips where the value lies within 2^-20 of a border
    assert ((out.double().cpu() - ref).abs() <= (u + 2.0 ** -18) * size + 1e-7).double().mean() >= 0.99
    ok = slots >= 0
    vr = torch.zeros_like(vc.cpu())
    Q.write(vr, v.cpu(), slots)
    same_bytes(vc, vr)                                   # values: exactly what the store puts there
    kref, knormed = norm_rotate(k.cpu(), kw, pos, rd, 1e-6, 1e6)
    ksize = knormed.abs() + torch.cat((knormed[..., rd // 2:rd], knormed[..., :rd // 2], 0 * knormed[..., rd:]), -1).abs()
    got = Q.read(kc, slots)[ok]
    _, scale, _ = Q.quantise(kref.to(dtype))
    # off by half a scale (a little more where the scale was rounded down), and by what the rotated key itself may be off
    # (its own group's ends as well, hence twice)
    step = scale.double()[ok].repeat_interleave(64, -1).flatten(-2).view(got.shape)
    limit = step * (0.5 + 16 * u) + (2 * (3 * u + 2.0 ** -19)) * ksize[ok].amax(-1, keepdim=True) + u * kref[ok].abs() + 1e-6
    assert ((got - kref[ok]).abs() <= limit).all()
    assert K.device_status() == (2 if n > 5 else 0)


# ------------------------------------------------------------------ attention
def sequences(gen, kv_lens, page_size, hkv, d, dtype, spread=1.0):
    """Pools filled through the store, and the pages of sequences of these lengths, in any order."""
    need = [-(-t // page_size) for t in kv_lens]
    total = sum(need) + 2
    order = torch.randperm(total, generator=gen)[:sum(need)].int()
    kc, vc = pools(total * page_size, hkv, d, dtype)
    every = torch.arange(total * page_size).int().cuda()
    K.store_kv_cache_q4(kc, vc, every, rows(gen, len(every), hkv, d, dtype, spread).cuda(),
                        rows(gen, len(every), hkv, d, dtype).cuda())
    indptr = torch.tensor([0] + need).cumsum(0).int()
    slots = [(order[indptr[b]:indptr[b + 1]].long()[:, None] * page_size + torch.arange(page_size)).flatten()[:t]
             for b, t in enumerate(kv_lens)]
    return kc, vc, indptr, order, slots


def assert_within(out, ref, weighted, size, dtype):
    """The output is rounded to the type, and in front of that in f16 (half a unit u16 = 2^-12, as f16 is what the products
    take): decode rounds weight times scale, p scale n <= p range, where n is the code and the range its group's; prefill rounds the weight and
    the value, p |v| each; `weighted` is the sum of the weights times the larger of |v| and the range.  A score is off by fp32
    accumulation (2^-20 of the sum of its terms' sizes covers 256 of them) and, in prefill, by u16 of it, as keys are rounded; where the sizes of terms are those of scale n and bias instead of their
    sum k, they are at most 2 range + |k| <= 31 |k| for all but keys near their group's zero: 2^-15 of the size."""
    u, u16 = half_unit(dtype), 2.0 ** -12
    score = size[..., None] * (u16 + 2.0 ** -15) + 2.0 ** -20
    tol = (2 * u16 + 2 * score.expm1()) * weighted + u * ref.abs() + 1e-6
    err = (out.double().cpu() - ref).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"{float((err / tol).max()):.3g} times the bound"
    # roundings are independent: as norms they are a fraction (1/sqrt 3) of half a unit each; u of the output, and of u16 four
    # with up to 2.5 times the output's size (the range against |v|)
    if ref.numel() > 4096 and ref.norm() > 0:
        rel = float((out.double().cpu() - ref).norm() / ref.norm())
        assert rel <= u / 3 ** 0.5 + 2.5 * 2 * u16, f"{rel:.3g} off as a norm"


DECODE = [
    # hq, hkv, d, dtype, page_size, lengths
    (16, 8, 128, BF16, 16, [1]),
    (16, 8, 128, F16, 16, [0, 1, 15, 16, 17, 0, 700]),
    (8, 8, 128, BF16, 32, [33, 257, 1000]),
    (32, 8, 128, F16, 16, [5000, 3, 129]),
    (40, 8, 128, BF16, 16, [300, 301]),
    (32, 2, 128, BF16, 64, [900, 64, 65]),
    (36, 3, 128, F16, 16, [77, 2000]),
    (16, 2, 256, F16, 16, [4000, 0, 31]),
    (24, 4, 256, BF16, 16, [513, 100, 1]),
    (32, 2, 256, BF16, 48, [700, 47, 49]),
    (13, 1, 256, F16, 16, [1234]),
    (1, 1, 128, BF16, 16, [20000]),
]


@pytest.mark.parametrize("hq,hkv,d,dtype,page_size,kv_lens", DECODE)
@pytest.mark.parametrize("gated", [False, True])
def test_decode(hq, hkv, d, dtype, page_size, kv_lens, gated):
    clean()
    gen = torch.Generator().manual_seed(hq + d + len(kv_lens))
    kc, vc, indptr, order, slots = sequences(gen, kv_lens, page_size, hkv, d, dtype)
    q = torch.randn(len(kv_lens), hq, d, generator=gen).to(dtype)
    gate = torch.randn(len(kv_lens), hq, d, generator=gen).to(dtype) if gated else None
    scale = 1 / math.sqrt(d)
    args = (q.cuda(), kc, vc, indptr.cuda(), order.cuda(), torch.tensor(kv_lens).int().cuda(), scale)
    out = K.paged_decode_attention_q4(*args, page_size=page_size, gate=None if gate is None else gate.cuda())
    parts = [Q.attention(q[b:b + 1], kc, vc, s, torch.ones(1, len(s), dtype=torch.bool), scale) for b, s in enumerate(slots)]
    ref, weighted, size = (torch.cat(x) for x in zip(*parts))
    if gated:      # (both factors rounded, and the product: another two half units)
        g = torch.sigmoid(gate.double())
        err = (out.double().cpu() - ref * g).abs()
        plain = K.paged_decode_attention_q4(*args, page_size=page_size)
        u = half_unit(dtype)
        assert (err <= (plain.double().cpu() - ref).abs() * g * (1 + 4 * u) + 2.1 * u * (ref * g).abs() + 1e-6).all()
    else:
        assert_within(out, ref, weighted, size, dtype)
        for b, t in enumerate(kv_lens):
            if t == 0:
                assert (out[b] == 0).all()
    # the same call gives the same bits
    again = K.paged_decode_attention_q4(*args, page_size=page_size, gate=None if gate is None else gate.cuda())
    assert torch.equal(out, again)
    clean()


PREFILL = [
    # hq, hkv, d, dtype, page_size, cached, new, cross, window
    (16, 8, 128, BF16, 16, [0], [1], False, 0),
    (16, 8, 128, F16, 16, [0, 5, 300], [17, 1, 40], False, 0),
    (32, 4, 128, BF16, 32, [1000, 50, 2000], [8, 8, 8], False, 0),
    (32, 8, 128, BF16, 16, [700, 900], [16, 16], True, 256),
    (32, 8, 128, F16, 16, [100, 0, 31], [200, 333, 70], False, 0),
    (8, 8, 128, BF16, 16, [64], [500], False, 100),
    (40, 8, 128, BF16, 16, [129, 3], [60, 90], False, 0),
    (16, 2, 256, F16, 16, [513], [100], False, 0),
    (24, 4, 256, BF16, 16, [0, 1000], [77, 5], False, 0),
    (32, 2, 256, BF16, 64, [40], [30], True, 0),
    (6, 2, 128, F16, 16, [9000], [3], False, 0),
    (32, 4, 128, BF16, 16, [4000], [130], False, 1024),
]


# long ones, most of which expand their pages first
LONG = [
    (32, 8, 128, BF16, 16, [4000], [2100], False, 0),
    (32, 4, 128, F16, 32, [3001, 500], [1800, 1500], False, 0),
    (16, 4, 256, BF16, 16, [2500], [1900], False, 1500),
    (24, 2, 256, F16, 16, [700, 1], [1333, 2000], True, 0),
    (40, 8, 128, BF16, 16, [5000], [1700], False, 0),
]


def test_long_prefills_expand_their_pages():
    def expanded(hq, hkv, d, dtype, page_size, cached, new, cross, window):
        pages = sum(-(-(a + b) // page_size) for a, b in zip(cached, new))
        return _lib.lib().msgl_prefill_expanded_bytes_q4(len(new), sum(new), pages, page_size, hq, hkv, d, int(dtype == F16),
                                                         max(new), cross, window)

    assert sum(expanded(*case) > 0 for case in LONG) >= 3
    assert not any(expanded(*case) for case in PREFILL)


def mask_of(cached, new, cross, window):
    pos = (cached + torch.arange(new))[:, None]
    t = torch.arange(cached + new)
    seen = (t <= pos) | cross
    return seen & (t >= pos - window + 1) if window else seen


@pytest.mark.parametrize("hq,hkv,d,dtype,page_size,cached,new,cross,window", PREFILL + LONG)
def test_prefill(hq, hkv, d, dtype, page_size, cached, new, cross, window):
    clean()
    long = sum(new) > 1500
    gen = torch.Generator().manual_seed(hq * d + sum(new))
    kv_lens = [a + b for a, b in zip(cached, new)]
    kc, vc, indptr, order, slots = sequences(gen, kv_lens, page_size, hkv, d, dtype)
    q = torch.randn(sum(new), hq, d, generator=gen).to(dtype)
    scale = 1 / math.sqrt(d)
    qo = torch.tensor([0] + new).cumsum(0).int()

    def ints(x):
        return torch.tensor(x).int().cuda()

    def call(**kw):
        return K.paged_prefill_attention_q4(q.cuda(), kc, vc, qo.cuda(), indptr.cuda(), order.cuda(), ints(kv_lens),
                                            ints(cached), scale, max(new), page_size=page_size, is_cross_attention=cross,
                                            sliding_window_size=window, **kw)

    out = call()
    parts = [Q.attention(q[qo[b]:qo[b + 1]], kc, vc, s, mask_of(cached[b], new[b], cross, window), scale,
                         "cuda" if long else "cpu") for b, s in enumerate(slots)]
    ref, weighted, size = (torch.cat(x) for x in zip(*parts))
    assert_within(out, ref, weighted, size, dtype)
    gate = torch.randn(q.shape, generator=gen).to(dtype)
    g = torch.sigmoid(gate.double())
    u = half_unit(dtype)
    err = (call(gate=gate.cuda()).double().cpu() - ref * g).abs()
    assert (err <= (out.double().cpu() - ref).abs() * g * (1 + 4 * u) + 2.1 * u * (ref * g).abs() + 1e-6).all()
    assert torch.equal(out, call())
    clean()
