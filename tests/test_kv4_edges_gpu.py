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
        assert (got == tiles) == (batch > 65535)


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
