"""Calls at the edges of what the 4-bit pool's operators take."""
import math

import pytest
import torch

from mini_sglang_mlx_b200 import _lib
from mini_sglang_mlx_b200 import kernel as K
from oracle import kv4_oracle as Q
from tests.test_kv4_gpu import BF16, F16, assert_within, mask_of, pools, rows, sequences


def ints(x):
    return torch.as_tensor(x).int().cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 128), (8, 4, 256), (16, 1, 128)])
def test_a_pool_without_slots(hq, hkv, d):
    """Through the C ABI: no slots, no pages, nothing but empty sequences: rows of zeros."""
    lib = _lib.lib()
    q = torch.ones(3, hq, d, dtype=BF16, device="cuda")
    some = torch.zeros(64, dtype=BF16, device="cuda")           # (a pointer that nothing is read through)
    stream = torch.cuda.current_stream().cuda_stream
    nbytes = lib.msgl_decode_workspace_bytes_q4(3, hq, hkv, d, 0, 16)
    ws = torch.zeros(nbytes, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, math.nan)
    zeros = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert lib.msgl_paged_decode_attention_q4(q.data_ptr(), some.data_ptr(), some.data_ptr(), zeros.data_ptr(), None, zeros.data_ptr(),
                                              None, out.data_ptr(), ws.data_ptr(), nbytes, 3, hq, hkv, d, 0, 0, 0.1, 16, 0, stream) == 0
    torch.cuda.synchronize()
    assert (out == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 2])
def test_row_pointers_that_fit_no_batch_give_zeros(new):
    """(One call's workspace is the next one's: what is right afterwards shows that nothing was left in it.)"""
    batch, pages = 16384, 4096
    kc, vc = pools(pages * 16, 1, 128, BF16, fill=0x3c)
    ends = ints([0, pages] * (batch // 2) + [0])
    ids = torch.zeros(pages, dtype=torch.int32, device="cuda")
    lens = torch.full((batch,), 1 << 20, dtype=torch.int32, device="cuda")
    q = torch.ones(batch * new, 1, 128, dtype=BF16, device="cuda")
    for _ in range(2):
        dirt = torch.full_like(q, math.nan)          # (what the result's memory held)
        del dirt
        if new == 1:
            out = K.paged_decode_attention_q4(q, kc, vc, ends, ids, lens, 0.1, page_size=256)
        else:
            out = K.paged_prefill_attention_q4(q, kc, vc, torch.arange(0, batch * new + 1, new).int().cuda(), ends, ids, lens,
                                               lens - new, 0.1, new, page_size=256)
        assert K.device_status() == 2 and (out == 0).all()


def test_workspace_of_a_batch_beyond_the_decode_kernels():
    """More sequences than a grid of the decode kernel numbers go to the tile kernel: its workspace, whatever the block's columns."""
    lib = _lib.lib()
    for batch in (65535, 65536, 70000):
        got = lib.msgl_prefill_workspace_bytes_q4(batch, batch, batch, 16, 16, 2, 128, 1, 0)
        tiles = lib.msgl_prefill_workspace_bytes(batch, batch, batch * 16, 16, 2, 128, 1, 0)
        tops = batch * 2 * 64 * 4                      # (the largest numbers of every sequence and head, behind what the tile kernel takes)
        assert (0 <= got - tiles - tops < 256) == (batch > 65535)


@pytest.mark.gpu
def test_prefill_of_more_sequences_than_the_decode_kernel_numbers():
    gen = torch.Generator().manual_seed(41)
    batch = 66000
    lens = [1 + i % 5 for i in range(batch)]
    kc, vc, indptr, order, slots = sequences(gen, lens, 16, 1, 128, BF16)
    q = torch.randn(batch, 2, 128, generator=gen).to(BF16)
    out = K.paged_prefill_attention_q4(q.cuda(), kc, vc, torch.arange(batch + 1).int().cuda(), ints(indptr), ints(order), ints(lens),
                                       ints(lens) - 1, 0.09, 1)
    for b in (0, 1, 65534, 65535, 65536, batch - 1):
        assert_within(out[b:b + 1], *Q.attention(q[b:b + 1], kc, vc, slots[b], torch.ones(1, lens[b], dtype=torch.bool), 0.09), BF16)
    assert K.device_status() == 0


BLOCKS = [
    # hq, hkv, d, dtype, page_size, cached, new
    (8, 8, 128, BF16, 16, [700, 33], [5, 16]),
    (16, 4, 128, F16, 16, [0, 1000, 17], [1, 4, 3]),
    (32, 8, 128, BF16, 32, [2000, 300], [4, 4]),
    (8, 4, 256, BF16, 16, [500, 3], [2, 8]),
    (16, 2, 256, F16, 64, [90, 4000], [2, 2]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,dtype,page_size,cached,new", BLOCKS)
@pytest.mark.parametrize("cross,window", [(False, 1), (False, 3), (False, 40), (False, 5000), (True, 0), (True, 40), (True, 2)])
@pytest.mark.parametrize("gated", [False, True])
def test_masks_of_short_blocks(hq, hkv, d, dtype, page_size, cached, new, cross, window, gated):
    """Up to sixteen rows a KV head run the decode kernel: sliding windows and bidirectional masks against 64 bits."""
    assert max(new) * hq // hkv <= 16
    gen = torch.Generator().manual_seed(hq + d + window)
    lens = [a + b for a, b in zip(cached, new)]
    kc, vc, indptr, order, slots = sequences(gen, lens, page_size, hkv, d, dtype)
    q = torch.randn(sum(new), hq, d, generator=gen).to(dtype)
    gate = torch.randn(q.shape, generator=gen).to(dtype) if gated else None
    qo = torch.tensor([0] + new).cumsum(0).int()

    def call(gate):
        return K.paged_prefill_attention_q4(q.cuda(), kc, vc, ints(qo), ints(indptr), ints(order), ints(lens), ints(cached), 0.09, max(new),
                                            page_size=page_size, is_cross_attention=cross, sliding_window_size=window, gate=gate)

    plain = call(None)
    parts = [Q.attention(q[qo[b]:qo[b + 1]], kc, vc, s, mask_of(cached[b], new[b], cross, window), 0.09) for b, s in enumerate(slots)]
    ref, weighted, size = (torch.cat(x) for x in zip(*parts))
    assert_within(plain, ref, weighted, size, dtype)
    if gated:      # (the output, the sigmoid and the product are rounded: three half units; one is in `plain`)
        g, u = torch.sigmoid(gate.double()), torch.finfo(dtype).eps / 2
        err = (call(gate.cuda()).double().cpu() - ref * g).abs()
        assert (err <= (plain.double().cpu() - ref).abs() * g * (1 + 4 * u) + 2.1 * u * (ref * g).abs() + 1e-6).all()
    assert K.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("d,page_size", [(128, 16), (256, 32)])
def test_a_cached_prefix_over_4_bit_pages(d, page_size):
    """Prompts that share prefixes, through the radix cache: a request's new tokens attend to pages that another one filled."""
    from types import SimpleNamespace

    import numpy as np

    from mini_sglang_mlx_b200.attention import AttnBackend
    from mini_sglang_mlx_b200.core import Batch, BatchPhase, Req
    from mini_sglang_mlx_b200.kvcache import MHAKVCacheQ4
    from mini_sglang_mlx_b200.scheduler import CacheManager, TableManager

    gen = torch.Generator().manual_seed(43)
    hq, hkv, vocab, pages = 8, 2, 300, 80
    emb_q, emb_k, emb_v = (rows(gen, vocab, h, d, BF16) for h in (hq, hkv, hkv))
    pool = MHAKVCacheQ4(hkv, 1, d, pages * page_size, BF16)
    table = torch.zeros((5, 640), dtype=torch.int32, device="cuda")
    tm, cm = TableManager(4, table), CacheManager("cuda", pages, page_size=page_size)
    backend = AttnBackend(SimpleNamespace(head_dim=d, num_kv_heads=hkv), pool, table, page_size=page_size)
    rng = np.random.default_rng(3)
    shared = rng.integers(0, vocab, size=300).tolist()
    prompts = [shared[:200] + rng.integers(0, vocab, size=17).tolist(), shared[:150] + rng.integers(0, vocab, size=60).tolist(),
               shared[:200] + rng.integers(0, vocab, size=1).tolist(), shared[:150] + rng.integers(0, vocab, size=333).tolist()]
    reused = 0
    for tokens in prompts:
        n, t = len(tokens), torch.tensor(tokens)
        handle, cached = cm.match_req(SimpleNamespace(input_ids=np.asarray(tokens, dtype=np.int32), input_len=n))
        have = handle.cached_len
        reused += have
        cm.lock(handle)
        row = tm.allocate()
        table[row, :have] = cached
        fresh = cm.allocate(n - have, start=have)
        table[row, have:n] = fresh
        batch = Batch(reqs=[Req(table_idx=row, cached_len=have, device_len=n)], phase=BatchPhase.PREFILL, out_loc=fresh)
        backend.prepare_metadata(batch)
        out = backend.forward(*(e[t[have:]].cuda() for e in (emb_q, emb_k, emb_v)), 0, batch)
        own = [torch.zeros(K.kv_cache_q4_shape(n, hkv, d), dtype=BF16) for _ in range(2)]      # the whole prompt, in a pool of its own
        for p, e in zip(own, (emb_k, emb_v)):
            Q.write(p, e[t], range(n))
        assert_within(out, *Q.attention(emb_q[t[have:]], *own, torch.arange(n), mask_of(have, n - have, False, 0), backend.sm_scale), BF16)
        cm.free_and_cache_finished_req(handle, np.asarray(tokens, np.int32), table[row, :n])
        tm.free(row)
        cm.check_integrity()
    assert reused >= 400 and K.device_status() == 0
