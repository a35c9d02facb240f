"""The rotation in front of the 4-bit pool: a rounding that falls the other way costs a key a whole step of its group, so the chain is
held to separate fp32 operations over sines and cosines of 64 bits."""
import pytest
import torch

from mini_sglang_mlx_b200 import kernel as K
from oracle import kv4_oracle as Q
from tests.test_kv4_gpu import BF16, F16, pools

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,rd,base", [(128, 128, 1e6), (128, 64, 1e4), (256, 64, 1e7), (256, 256, 5e5), (128, 32, 1e6)])
@pytest.mark.parametrize("far", [1000, 200000, (1 << 24) - 1])
def test_rotation_is_that_of_fp32_operations(dtype, d, rd, base, far):
    """Sines are taken in 64 bits of an angle good to 2^-53 of itself and rounded to fp32: another neighbour with a probability of the angle's error
    over half a unit, 2^-53 far / 2^-25, doubled for the polynomials.  Of those, one in 2^12 (f16, 2^-24 over half of 2^-11) changes a result, and
    a key's element three: its own, and its group's ends.  The bound is four times that, and 2^-18 at least."""
    gen = torch.Generator(device="cuda").manual_seed(rd + far)
    n, hq, hkv = 4000, 4, 4
    qkv = (torch.randn(n, hq + 2 * hkv, d, generator=gen, device="cuda") * 3).to(dtype)
    q, k, v = qkv.split((hq, hkv, hkv), 1)
    pos = torch.randint(0, far + 1, (n,), generator=gen, device="cuda").int()
    slots = torch.randperm(n, generator=gen, device="cuda").int()
    kc, vc = pools(n, hkv, d, dtype)
    out = K.qk_norm_rope_store_q4(q, k, v, None, None, pos, slots, kc, vc, rope_base=base, rotary_dim=rd)
    half = rd // 2
    angle = pos.double()[:, None, None] * base ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    cos, sin = angle.cos().float(), angle.sin().float()

    def turned(x):
        a, b = x[..., :half].float(), x[..., half:rd].float()
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., rd:].float()), -1).to(dtype)

    share = max(2.0 ** -18, 4 * 2 * 2.0 ** -53 * far / 2.0 ** -25 * 2.0 ** -12 * 3)
    assert float((out != turned(q)).float().mean()) <= share
    at = torch.arange(n).int()
    want = torch.empty(n, hkv, d, dtype=torch.float64)
    want[slots.long().cpu()] = Q.values(*Q.quantise(turned(k).cpu()))
    assert float((Q.read(kc, at) != want).float().mean()) <= share
    assert K.device_status() == 0
