"""Reports of several kernels in one status word: none takes another's away."""
import ctypes
import math

import pytest
import torch

from mini_sglang_mlx_b200 import _lib
from mini_sglang_mlx_b200 import kernel as K
from tests.test_kv4_gpu import BF16, pools

pytestmark = pytest.mark.gpu


def store_what_is_not_finite():
    kc, vc = pools(16, 1, 128, BF16)
    rows = torch.full((1, 1, 128), math.nan, dtype=BF16, device="cuda")
    K.store_kv_cache_q4(kc, vc, torch.zeros(1, dtype=torch.int32, device="cuda"), rows, rows)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def store_16():
    pool = torch.zeros(16, 1, 128, dtype=BF16, device="cuda")
    row = torch.ones(1, 1, 128, dtype=BF16, device="cuda")
    K.store_kv_cache(pool, pool.clone(), ints(99), row, row)


def decode_16():
    pool = torch.zeros(32, 1, 128, dtype=BF16, device="cuda")
    K.paged_decode_attention_p16(torch.ones(1, 1, 128, dtype=BF16, device="cuda"), pool, pool, ints(0, 1), ints(7), ints(16), ints(1),
                                 0.1, 8)


def decode_16_length():
    pool = torch.zeros(32, 1, 128, dtype=BF16, device="cuda")
    K.paged_decode_attention_p16(torch.ones(1, 1, 128, dtype=BF16, device="cuda"), pool, pool, ints(0, 1), ints(0), ints(17), ints(1),
                                 0.1, 8)


@pytest.mark.parametrize("bad", [store_16, decode_16, decode_16_length])
def test_a_report_of_the_4_bit_pool_outlives_one_of_a_16_bit_pool(bad):
    K.device_status()
    for first, second in ((store_what_is_not_finite, bad), (bad, store_what_is_not_finite)):
        first()
        second()
        assert K.device_status() == 6
    assert K.device_status() == 0


def test_read_status_names_what_was_reported():
    lib = _lib.lib()
    ws = torch.zeros(1024, dtype=torch.uint8, device="cuda")
    word = ctypes.c_int(-1)
    stream = torch.cuda.current_stream().cuda_stream
    for value, texts in ((1, ["bounded wait"]), (2, ["outside the pool"]), (4, ["not finite"]), (6, ["outside the pool", "not finite"]),
                         (3, ["bounded wait", "outside the pool"]), (8, ["unknown device status 8"])):
        ws[:4].view(torch.int32).fill_(value)
        assert lib.msgl_read_status(ws.data_ptr(), 1, ctypes.byref(word), stream) == 7 and word.value == value
        for text in texts:
            assert text in _lib.last_error()
