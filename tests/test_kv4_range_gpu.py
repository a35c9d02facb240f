"""The 4-bit K/V pool over the whole range of its numbers: small and large rows, groups and tokens of very unlike size, in every form of
the attention, against 64 bits."""
import math

import pytest
import torch

from mini_sglang_mlx_b200 import _lib
from mini_sglang_mlx_b200 import kernel as K
from oracle import kv4_oracle as Q
from tests.test_kv4_gpu import BF16, F16, half_unit, mask_of, pools

pytestmark = pytest.mark.gpu

# hq, hkv, d, cached, new: the decode kernel (one token; a block), one CTA of 128 and of 256 rows, its key range split, pages expanded first
FORMS = {
    "decode": (16, 4, 128, [300, 45, 1000], [1, 1, 1]),
    "decode_16_heads": (16, 1, 128, [300, 45, 1000], [1, 1, 1]),
    "decode_256": (16, 2, 256, [300, 45, 700], [1, 1, 1]),
    "block": (8, 4, 128, [300, 45], [5, 5]),
    "one_cta": (16, 4, 128, [300, 45], [30, 22]),
    "one_cta_256": (16, 4, 256, [300, 45], [30, 22]),
    "one_cta_two_tiles": (16, 4, 128, [200, 45], [90, 150]),
    "one_cta_split": (16, 4, 128, [6000], [30]),
    "expanded": (32, 4, 128, [4000], [2100]),
    "expanded_256": (16, 2, 256, [900], [1500]),
}


class Call:
    """Pools that hold ``k`` and ``v`` (tokens of all sequences, heads, d) and a call over them."""

    def __init__(self, gen, form, dtype, k, v, page_size=16):
        self.hq, self.hkv, self.d, self.cached, self.new = FORMS[form]
        self.form, self.dtype, self.page_size = form, dtype, page_size
        self.lens = [a + b for a, b in zip(self.cached, self.new)]
        need = [-(-t // page_size) for t in self.lens]
        self.order = torch.randperm(sum(need) + 2, generator=gen)[:sum(need)].int()
        self.indptr = torch.tensor([0] + need).cumsum(0).int()
        self.slots = [(self.order[self.indptr[b]:self.indptr[b + 1]].long()[:, None] * page_size + torch.arange(page_size)).flatten()[:t]
                      for b, t in enumerate(self.lens)]
        self.kc, self.vc = pools((sum(need) + 2) * page_size, self.hkv, self.d, dtype)
        K.store_kv_cache_q4(self.kc, self.vc, torch.cat(self.slots).int().cuda(), k.to(dtype).cuda(), v.to(dtype).cuda())

    def __call__(self, q, scale, cross=False, window=0):
        def ints(x):
            return torch.tensor(x).int().cuda()

        if self.form.startswith("decode"):
            return K.paged_decode_attention_q4(q.cuda(), self.kc, self.vc, self.indptr.cuda(), self.order.cuda(), ints(self.lens), scale,
                                               page_size=self.page_size)
        return K.paged_prefill_attention_q4(q.cuda(), self.kc, self.vc, ints([0, *torch.tensor(self.new).cumsum(0).tolist()]),
                                            self.indptr.cuda(), self.order.cuda(), ints(self.lens), ints(self.cached), scale,
                                            max(self.new), page_size=self.page_size, is_cross_attention=cross,
                                            sliding_window_size=window)

    def reference(self, q, scale, cross=False, window=0):
        parts, a = [], 0
        for b, n in enumerate(self.new):
            parts.append(Q.attention(q[a:a + n], self.kc, self.vc, self.slots[b], mask_of(self.cached[b], n, cross, window), scale,
                                     "cuda" if sum(self.new) > 500 else "cpu"))
            a += n
        return [torch.cat(x) for x in zip(*parts)]


def tokens(form):
    return sum(FORMS[form][3]) + sum(FORMS[form][4])


def queries(gen, form, dtype, size=1.0):
    hq, _, d, _, new = FORMS[form]
    return (torch.randn(sum(new), hq, d, generator=gen) * size).to(dtype)


def assert_near(out, ref, weighted, size, dtype, keys):
    """Half a unit u of the output; half a unit u16 = 2^-11 of f16 of the weight (decode: weight times scale, with codes up to 15 scales =
    the range of the group; prefill: the weight times |v|), and of the value (prefill); scores are off by u16 of the size of their terms (keys, prefill)
    and by 2^-15 of it (fp32 sums of up to 31 times that size); weights below 2^-14 of the largest are off by 2^-25 of it, times 15 codes, `keys` of them.
    No absolute term: the bound goes with the values."""
    u, u16 = half_unit(dtype), half_unit(F16)
    tol = (2 * u16 + keys * 2.0 ** -21 + 2 * (size[..., None] * (u16 + 2.0 ** -15) + 2.0 ** -20).expm1()) * weighted + u * ref.abs()
    if dtype == F16:
        tol = tol + 2.0 ** -25                            # half a unit of a subnormal output
    err = (out.double().cpu() - ref).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"{float((err / tol.clamp(min=1e-300)).max()):.3g} times the bound"


def rel(out, ref):
    return float((out.double().cpu() - ref).norm() / ref.norm())


def test_the_forms_are_those_that_the_names_say():
    def expanded(hq, hkv, d, cached, new):
        pages = sum(-(-(a + b) // 16) for a, b in zip(cached, new))
        return _lib.lib().msgl_prefill_expanded_bytes_q4(len(new), sum(new), pages, 16, hq, hkv, d, 0, max(new), 0, 0) > 0

    for name, case in FORMS.items():
        assert expanded(*case) == name.startswith("expanded"), name


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype,size", [(BF16, 2e-28), (BF16, 3e-8), (BF16, 1e-5), (BF16, 3000.0), (F16, 3000.0), (F16, 1e-2)])
def test_small_and_large_keys_and_values(form, dtype, size):
    """Keys and values of one size, with scores of order 1."""
    gen = torch.Generator().manual_seed(21)
    _, hkv, d, _, _ = FORMS[form]
    n = tokens(form)
    call = Call(gen, form, dtype, torch.randn(n, hkv, d, generator=gen) * size, torch.randn(n, hkv, d, generator=gen) * size)
    q, scale = queries(gen, form, dtype), 0.09 / size
    out = call(q, scale)
    ref, weighted, terms = call.reference(q, scale)
    assert_near(out, ref, weighted, terms, dtype, max(call.lens))
    # as a norm: independent roundings, each 1/sqrt 3 of half a unit: the output's, and of f16 four with up to 2.5 times the output's
    # size (an element against the range of its group); a subnormal f16 output has half a unit of 2^-24
    tiny = 2.0 ** -25 / float(ref.abs().mean()) if dtype == F16 else 0.0
    assert rel(out, ref) <= half_unit(dtype) / 3 ** 0.5 + 2.5 * 4 * half_unit(F16) / 3 ** 0.5 + tiny
    assert K.device_status() == 0


@pytest.mark.parametrize("form", FORMS)
def test_powers_of_two_change_no_bit(form):
    """Values times a power of two give results times that power; keys and the scores' scale one up, the other down, the same."""
    gen = torch.Generator().manual_seed(22)
    _, hkv, d, _, _ = FORMS[form]
    n = tokens(form)
    k, v = torch.randn(n, hkv, d, generator=gen).to(BF16), torch.randn(n, hkv, d, generator=gen).to(BF16)
    q = queries(gen, form, BF16)
    want = None
    for a, b in ((0, 0), (0, -30), (-25, 0), (-60, -70), (11, 12)):
        state = gen.get_state()
        out = Call(gen, form, BF16, k.float() * 2.0 ** a, v.float() * 2.0 ** b)(q, 0.09 * 2.0 ** -a).float() * 2.0 ** -b
        gen.set_state(state)
        want = out if want is None else want
        assert torch.equal(out, want), (a, b)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype,spread", [(BF16, 2.0 ** -16), (BF16, 2.0 ** 12), (F16, 2.0 ** -8), (F16, 2.0 ** 10)])
def test_groups_of_unlike_size(form, dtype, spread):
    """The first 64 elements of every value are of order 1, the others of another: each is as good as it is alone."""
    gen = torch.Generator().manual_seed(23)
    _, hkv, d, _, _ = FORMS[form]
    n = tokens(form)
    v = torch.randn(n, hkv, d, generator=gen)
    v[..., 64:] *= spread
    call = Call(gen, form, dtype, torch.randn(n, hkv, d, generator=gen), v)
    q = queries(gen, form, dtype)
    out = call(q, 0.09)
    ref, weighted, terms = call.reference(q, 0.09)
    assert_near(out, ref, weighted, terms, dtype, max(call.lens))
    for part in (slice(0, 64), slice(64, d)):
        tiny = 2.0 ** -25 / float(ref[..., part].abs().mean()) if dtype == F16 else 0.0
        assert rel(out[..., part], ref[..., part]) <= half_unit(dtype) / 3 ** 0.5 + 2.5 * 4 * half_unit(F16) / 3 ** 0.5 + tiny


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("score", [-60.0, -12.0, 0.0])
def test_one_huge_value(form, dtype, score):
    """A token whose value is 2^21 times the others': of next to no weight (2^-60, 2^-12 of an ordinary key's) or of theirs."""
    gen = torch.Generator().manual_seed(24)
    _, hkv, d, _, _ = FORMS[form]
    n = tokens(form)
    k, v = torch.randn(n, hkv, d, generator=gen), torch.randn(n, hkv, d, generator=gen) * 0.01
    k[..., 0] = 0.0
    for at in (7, 200):
        v[at] = torch.sign(v[at]) * 20000.0
        k[at] = 0.0
        k[at, :, 0] = 8 * score
    q = queries(gen, form, dtype)
    q[..., 0] = 1.0
    scale = math.log(2.0) / 8
    call = Call(gen, form, dtype, k, v)
    out = call(q, scale)
    ref, weighted, terms = call.reference(q, scale)
    # (the outlying key's own terms are exact: one element of q and k each)
    assert_near(out, ref, weighted, terms.clamp(max=25.0), dtype, max(call.lens))
    assert K.device_status() == 0


@pytest.mark.parametrize("form", [f for f in FORMS if not f.startswith("decode")])
@pytest.mark.parametrize("window", [0, 20])
def test_huge_values_that_a_row_does_not_see(form, window):
    """Values behind a row's position, or in front of its window, 2^21 times those that it sees."""
    gen = torch.Generator().manual_seed(25)
    hq, hkv, d, cached, new = FORMS[form]
    n = tokens(form)
    v = torch.randn(n, hkv, d, generator=gen) * 0.01
    ends = torch.tensor([a + b for a, b in zip(cached, new)]).cumsum(0)
    for e, b in zip(ends.tolist(), new):
        v[e - 1] *= 2.0 ** 21                              # the last token: only the last row sees it
        if window:
            v[e - b - window + 1] *= 2.0 ** 21             # the first token's window begins here: the second does not see it
    call = Call(gen, form, BF16, torch.randn(n, hkv, d, generator=gen), v.clamp(-30000, 30000))
    q = queries(gen, form, BF16)
    out = call(q, 0.09, window=window)
    ref, weighted, terms = call.reference(q, 0.09, window=window)
    assert_near(out, ref, weighted, terms, BF16, max(call.lens))
    assert K.device_status() == 0
