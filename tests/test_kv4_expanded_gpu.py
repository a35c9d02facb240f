"""Long prefills over a 4-bit pool, which expand their pages first: what stands in the index list and the pool beside the sequences' tokens."""
import math

import pytest
import torch

from mini_sglang_mlx_b200 import _lib
from mini_sglang_mlx_b200 import kernel as K
from oracle import kv4_oracle as Q
from tests.test_kv4_gpu import BF16, assert_within, mask_of, pools, rows

pytestmark = pytest.mark.gpu

# hq, hkv, d, cached, new
SHAPES = [(32, 4, 128, [8000, 8000], [2100, 2100]), (16, 2, 256, [900, 90], [1500, 150])]
OUTSIDE = 1 << 20


def ints(x):
    return torch.as_tensor(x).int().cuda()


class Batch:
    """Two sequences over pools of ``extra`` blocks more."""

    def __init__(self, shape, page_size=16, extra=2):
        gen = torch.Generator().manual_seed(31)
        self.hq, self.hkv, self.d, self.cached, self.new = shape
        self.page_size = page_size
        self.lens = [a + b for a, b in zip(self.cached, self.new)]
        need = [-(-t // page_size) for t in self.lens]
        self.order = torch.randperm(sum(need), generator=gen).int()
        self.indptr = torch.tensor([0] + need).cumsum(0).int()
        num_slots = sum(need) * page_size + 16 * extra
        self.kc, self.vc = pools(num_slots, self.hkv, self.d, BF16)
        every = torch.arange(num_slots).int().cuda()
        K.store_kv_cache_q4(self.kc, self.vc, every, *(rows(gen, num_slots, self.hkv, self.d, BF16).cuda() for _ in range(2)))
        self.q = torch.randn(sum(self.new), self.hq, self.d, generator=gen).to(BF16)
        assert K.device_status() == 0
        assert _lib.lib().msgl_prefill_expanded_bytes_q4(2, sum(self.new), sum(need), page_size, self.hq, self.hkv, self.d, 0,
                                                         max(self.new), 0, 0) > 0

    def __call__(self, order=None, kc=None, vc=None, lens=None, **kw):
        return K.paged_prefill_attention_q4(
            self.q.cuda(), self.kc if kc is None else kc, self.vc if vc is None else vc, ints([0, self.new[0], sum(self.new)]),
            ints(self.indptr), ints(self.order if order is None else order), ints(self.lens if lens is None else lens), ints(self.cached),
            0.09, self.new[0], page_size=self.page_size, **kw)

    def reference(self, order, cross=False, window=0):
        parts, a = [], 0
        for b, n in enumerate(self.new):
            pages = order[self.indptr[b]:self.indptr[b + 1]].long()
            slots = (pages[:, None] * self.page_size + torch.arange(self.page_size)).flatten()[:self.lens[b]]
            parts.append(Q.attention(self.q[a:a + n], self.kc, self.vc, slots, mask_of(self.cached[b], n, cross, window), 0.09, "cuda"))
            a += n
        return [torch.cat(x) for x in zip(*parts)]


@pytest.mark.parametrize("shape", SHAPES)
def test_entries_that_no_token_stands_in(shape):
    """Entries behind the last sequence's, and those of a sequence behind its length, hold anything; neither is read or reported."""
    b = Batch(shape)
    want = b()
    slack = torch.cat((b.order, torch.tensor([-1, OUTSIDE, -(1 << 30)]).int()))
    assert torch.equal(b(slack), want) and K.device_status() == 0
    lens = [b.lens[0] - 100, b.lens[1]]
    want = b(lens=lens)
    short = b.order.clone()
    short[-(-lens[0] // 16):b.indptr[1]] = -1
    assert torch.equal(b(short, lens=lens), want) and K.device_status() == 0


@pytest.mark.parametrize("shape", SHAPES)
def test_pages_in_front_of_the_window(shape):
    """Pages that no row's window reaches may be gone."""
    b = Batch(shape)
    window = 256
    want = b(sliding_window_size=window)
    gone = b.order.clone()
    for i, cached in enumerate(b.cached):
        gone[b.indptr[i]:b.indptr[i] + max(0, cached - window + 1) // 128 * 8] = -1
    assert (gone < 0).any()
    assert torch.equal(b(gone, sliding_window_size=window), want) and K.device_status() == 0


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("page_size", [16, 32])
@pytest.mark.parametrize("window", [0, 700])
def test_pages_outside_the_pool(shape, page_size, window):
    """A page outside the pool reads as zero keys and values and is reported; so is the part of the last page that lies outside."""
    b = Batch(shape, page_size, extra=1)
    order = b.order.clone()
    last = b.kc.shape[0] * 16 // page_size           # with pages of 32, half of it is there
    for at, page in ((-1, OUTSIDE), (b.indptr[1] - 3, -5), (b.indptr[1] - 9, last)):
        order[at] = page
    out = b(order, sliding_window_size=window)
    assert K.device_status() == 2
    assert_within(out, *b.reference(order, window=window), BF16)
    assert torch.equal(b(), b()) and K.device_status() == 0


@pytest.mark.parametrize("shape", SHAPES)
def test_lengths_beyond_the_pages(shape):
    b = Batch(shape)
    held = [16 * int(b.indptr[1]), 16 * int(b.indptr[2] - b.indptr[1])]
    want = b(lens=held)
    assert K.device_status() == 0
    assert torch.equal(b(lens=[10 ** 6, held[1]]), want)
    assert K.device_status() == 2


@pytest.mark.parametrize("shape", SHAPES)
def test_garbage_beside_the_tokens(shape):
    """Rows behind a sequence's last token and pages of nobody hold bytes that stand for NaN and infinity."""
    b = Batch(shape)
    want = [b(**kw) for kw in ({}, dict(is_cross_attention=True), dict(sliding_window_size=300))]
    used = torch.zeros(b.kc.shape[0] * 16, dtype=torch.bool)
    for i, n in enumerate(b.lens):
        pages = b.order[b.indptr[i]:b.indptr[i + 1]].long()
        used[(pages[:, None] * 16 + torch.arange(16)).flatten()[:n]] = True
    assert not used.all()
    dirty = []
    for pool, what in ((b.kc, math.nan), (b.vc, math.inf)):
        bad = torch.full_like(pool, what)
        x, y = (t.view(torch.uint8).view(-1, 9 * b.d) for t in (pool, bad))
        rows_of = used.view(-1, 1, 16).expand(-1, b.hkv, 16).reshape(-1, 16).cuda()
        for at, width in ((0, b.d // 2), (8 * b.d, b.d // 16)):
            src = x[:, at:at + 16 * width].reshape(-1, 16, width)
            dst = y[:, at:at + 16 * width].reshape(-1, 16, width)
            y[:, at:at + 16 * width] = torch.where(rows_of[..., None], src, dst).flatten(1)
        dirty.append(bad)
    got = [b(kc=dirty[0], vc=dirty[1], **kw) for kw in ({}, dict(is_cross_attention=True), dict(sliding_window_size=300))]
    for a, c in zip(got, want):
        assert torch.isfinite(a).all() and torch.equal(a, c)
    assert K.device_status() == 0
