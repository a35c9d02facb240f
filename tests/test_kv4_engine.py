"""The 4-bit pool where it is used: pool, allocator and attention backend together, streams, graphs, devices; and what the operators
refuse."""
import math
import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from mini_sglang_mlx_b200 import _lib
from mini_sglang_mlx_b200 import kernel as K
from mini_sglang_mlx_b200.attention import AttnBackend
from mini_sglang_mlx_b200.core import Batch, BatchPhase, Req
from mini_sglang_mlx_b200.kvcache import MHAKVCacheQ4
from mini_sglang_mlx_b200.scheduler import CacheManager, TableManager
from oracle import kv4_oracle as Q
from tests.test_kv4_gpu import BF16, F16, assert_within, half_unit, mask_of, norm_rotate, rows, sequences

ROOT = Path(__file__).resolve().parent.parent


# ------------------------------------------------------------------ on the CPU: shapes and refusals of the C ABI
def test_shape_of_a_pool():
    assert K.kv_cache_q4_shape(33, 4, 256) == (3, 4, 1152)
    assert K.kv_cache_q4_shape(0, 1, 128) == (0, 1, 576)
    for bad in ((16, 4, 64), (-1, 4, 128), (16, 0, 128)):
        with pytest.raises(RuntimeError, match="kv_cache_q4_shape"):
            K.kv_cache_q4_shape(*bad)


def test_quantised_values_are_within_half_a_scale():
    gen = torch.Generator().manual_seed(3)
    for dtype in (BF16, F16):
        x = rows(gen, 50, 3, 128, dtype, 5.0)
        codes, scale, bias = Q.quantise(x)
        off = (Q.values(codes, scale, bias) - x.double()).abs().unflatten(-1, (-1, 64))
        # half a scale; the top of a group also by what rounding took off 15 scales
        assert (off <= scale.double()[..., None] * (0.5 + 15 * half_unit(dtype))).all()
        pool = torch.zeros(K.kv_cache_q4_shape(64, 3, 128), dtype=dtype)
        slots = torch.randperm(64, generator=gen)[:50]
        Q.write(pool, x, slots.tolist())
        assert torch.equal(Q.read(pool, slots), Q.values(codes, scale, bias))


NULL = [None] * 9


def call(name, **kw):
    """An operator of the C ABI on null pointers: whatever it refuses, it refuses before it touches one."""
    a = dict(n=4, hq=16, hkv=8, d=128, slots=64, dtype=0, page=16, pages=4, rd=128, base=1e6, eps=1e-6, kstride=1024, window=0,
             batch=2)
    a.update(kw)
    lib = _lib.lib()
    if name == "store":
        return lib.msgl_store_kv_cache_q4(*NULL[:5], a["n"], a["hkv"], a["d"], a["slots"], a["kstride"], 1024, a["dtype"], None, None)
    if name == "load":
        return lib.msgl_load_kv_cache_q4(*NULL[:5], a["n"], a["hkv"], a["d"], a["slots"], a["dtype"], None, None)
    if name == "project":
        return lib.msgl_qk_norm_rope_store_q4(*NULL, None, a["n"], a["hq"], a["hkv"], a["d"], a["rd"], a["base"], a["eps"],
                                              a["slots"], 4096, a["kstride"], 1024, a["dtype"], None, None)
    if name == "decode":
        return lib.msgl_paged_decode_attention_q4(*NULL, 0, a["n"], a["hq"], a["hkv"], a["d"], a["slots"], a["dtype"], 0.1,
                                                  a["page"], a["pages"], None)
    return lib.msgl_paged_prefill_attention_q4(*NULL, None, None, 0, None, 0, a["batch"], a["n"], a["hq"], a["hkv"], a["d"],
                                               a["slots"], a["dtype"], 0.1, 2, 0, a["window"], a["page"], a["pages"], None)


EVERY = ("store", "load", "project", "decode", "prefill")


@pytest.mark.parametrize("names,kw,code,text", [
    (EVERY, dict(d=64), 3, "head_dim must be 128 or 256"),
    (EVERY, dict(dtype=7), 2, "unsupported dtype"),
    (EVERY, dict(slots=24), 1, "multiple of 16"),
    (EVERY, dict(slots=1 << 31), 1, "below 2^31"),
    (EVERY, dict(slots=(1 << 31) - 16, hkv=17), 1, "too many rows"),
    (EVERY, dict(hkv=0), 1, ""),
    (EVERY, dict(n=-1), 1, ""),
    (EVERY, dict(), 5, "null tensor pointer"),
    (("store", "project"), dict(kstride=1000), 1, "stride"),
    (("project",), dict(rd=96), 5, "rotary_dim"),
    (("project",), dict(base=1.0), 5, "rope_base"),
    (("project",), dict(eps=-1.0), 5, "eps"),
    (("decode", "prefill"), dict(hq=12), 4, "multiple of num_kv_heads"),
    (("decode",), dict(hq=34, hkv=2), 4, "<= 16"),
    (("decode", "prefill"), dict(page=8), 5, "page_size must be a multiple of 16"),
    (("decode", "prefill"), dict(page=0), 5, "page_size"),
    (("decode", "prefill"), dict(pages=1 << 28, page=16), 1, "2^31"),
    (("decode",), dict(n=70000), 1, "65535"),
    (("prefill",), dict(window=-1), 5, "sliding_window_size"),
    (("prefill",), dict(batch=0), 1, "batch must be > 0"),
])
def test_refusals_of_the_c_abi(names, kw, code, text):
    for name in names:
        assert call(name, **kw) == code, name
        assert text in _lib.last_error()


def test_empty_calls_of_the_c_abi():
    for name in EVERY:
        assert call(name, n=0) == 0


FAKE = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from mini_sglang_mlx_b200 import kernel as K
with FakeTensorMode():
    def new(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda:0")
    q, kc, k = new(1, 2, 128), new(4, 1, 576), new(1, 1, 128)
    two, one = new(2, dtype=torch.int32), new(1, dtype=torch.int32)
calls = [
    lambda: K.store_kv_cache_q4(kc, kc, one, k, k),
    lambda: K.load_kv_cache_q4(kc, kc, one),
    lambda: K.qk_norm_rope_store_q4(q, k, k, None, None, one, one, kc, kc, rope_base=1e6),
    lambda: K.paged_decode_attention_q4(q, kc, kc, two, one, one, 0.1),
    lambda: K.paged_prefill_attention_q4(q, kc, kc, two, two, one, one, one, 0.1, 1),
]
for call in calls:
    try:
        call()
    except RuntimeError:
        print("raised", flush=True)
"""


def test_what_cpp_throws_is_raised_and_does_not_end_the_process():
    proc = subprocess.run([sys.executable, "-c", FAKE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stderr[-2000:]
    assert proc.stdout.split() == ["raised"] * 5


def test_refusals_of_the_python_operators():
    """(On the CPU every call is declined by the native side, and the wrapper says why.)"""
    kc = torch.zeros(4, 2, 576, dtype=BF16)
    k = torch.zeros(3, 2, 128, dtype=BF16)
    q = torch.zeros(3, 4, 128, dtype=BF16)
    i3, i4 = torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for f in (lambda: K.store_kv_cache_q4(kc, kc, i3, k, k), lambda: K.load_kv_cache_q4(kc, kc, i3),
              lambda: K.qk_norm_rope_store_q4(q, k, k, None, None, i3, i3, kc, kc, rope_base=1e6),
              lambda: K.paged_decode_attention_q4(q, kc, kc, i4, i3, i3, 0.1),
              lambda: K.paged_prefill_attention_q4(q, kc, kc, i4, i4, i3, i3, i3, 0.1, 1)):
        with pytest.raises(RuntimeError, match="CUDA device"):
            f()
    for bad in (kc[..., :512], kc.float(), kc.transpose(0, 1), kc[0]):
        with pytest.raises(RuntimeError, match="load_kv_cache_q4: "):
            K.load_kv_cache_q4(bad, bad, i3)
    with pytest.raises(RuntimeError, match="v_cache must match"):
        K.load_kv_cache_q4(kc, kc[:2], i3)
    cfg = SimpleNamespace(head_dim=128, num_kv_heads=2)
    pool = MHAKVCacheQ4(2, 1, 128, 40, BF16, device="cpu")
    assert pool.num_pages == 48 and pool.num_layers == 1 and pool.dtype == BF16
    with pytest.raises(ValueError, match="multiple of 16"):
        AttnBackend(cfg, pool, torch.zeros(1, 64, dtype=torch.int32), page_size=8)
    with pytest.raises(ValueError, match="shape mismatch"):
        pool.store_kv(k, k, i4, 0)


# ------------------------------------------------------------------ on the GPU
@pytest.mark.gpu
def test_refusals_on_the_gpu():
    kc = torch.zeros(4, 2, 576, dtype=BF16, device="cuda")
    k = torch.zeros(3, 2, 128, dtype=BF16, device="cuda")
    q = torch.zeros(3, 4, 128, dtype=BF16, device="cuda")
    i3, i4 = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (3, 4))
    bad = [
        (lambda: K.store_kv_cache_q4(kc, kc, i3.long(), k, k), "int32"),
        (lambda: K.store_kv_cache_q4(kc, kc, i4, k, k), r"k must be \(4, 2, 128\)"),
        (lambda: K.store_kv_cache_q4(kc, kc, i3, k.half(), k), "pools' dtype"),
        (lambda: K.store_kv_cache_q4(kc, kc, i3, k.transpose(0, 1).contiguous().transpose(0, 1), k), "dense"),
        (lambda: K.store_kv_cache_q4(kc, kc, i3, k.cpu(), k), "same device"),
        (lambda: K.store_kv_cache_q4(kc, kc, i3, torch.zeros(3 * 256 + 2, dtype=BF16, device="cuda")[2:].view(3, 2, 128), k),
         "8-byte aligned"),
        (lambda: K.load_kv_cache_q4(kc[:, :1], kc[:, :1], i3), "contiguous"),
        (lambda: K.qk_norm_rope_store_q4(q, k, k, torch.ones(64, dtype=BF16, device="cuda"), None, i3, i3, kc, kc, rope_base=1e6),
         "norm weight"),
        (lambda: K.qk_norm_rope_store_q4(q, k, k, None, None, i4, i3, kc, kc, rope_base=1e6), "positions"),
        (lambda: K.qk_norm_rope_store_q4(q, k, k, None, None, i3, i3, kc, kc, rope_base=1e6, rotary_dim=48), "rotary_dim"),
        (lambda: K.paged_decode_attention_q4(q, kc, kc, i3, i3, i3, 0.1), "page_indptr must have 4"),
        (lambda: K.paged_decode_attention_q4(q, kc, kc, i4, i3, i3, 0.1, page_size=24), "multiple of 16"),
        (lambda: K.paged_decode_attention_q4(q, kc, kc, i4, i3, i3, 0.1, gate=q.half()), "gate"),
        (lambda: K.paged_decode_attention_q4(q[:, :3], kc, kc, i4, i3, i3, 0.1), "contiguous"),
        (lambda: K.paged_decode_attention_q4(q[:, :3].contiguous(), kc, kc, i4, i3, i3, 0.1), "multiple of num_kv_heads"),
        (lambda: K.paged_prefill_attention_q4(q, kc, kc, i4, i4, i3, i4, i3, 0.1, 1), "kv_lens must have 3"),
        (lambda: K.paged_prefill_attention_q4(q, kc, kc, i4, i4, i3, i3, i3, 0.1, 1, sliding_window_size=-2), "sliding_window_size"),
    ]
    for f, text in bad:
        with pytest.raises(RuntimeError, match=text):
            f()
    assert K.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("new,hq,hkv,d,window", [(1, 16, 8, 128, 0), (3, 16, 4, 128, 0), (40, 32, 4, 128, 20), (5, 16, 2, 256, 0)])
def test_pages_and_lengths_outside_the_pool(new, hq, hkv, d, window):
    """A page that is not in the pool reads as zero keys and values, a length beyond a sequence's pages is clamped; both are
    reported, and other sequences are as they were."""
    gen = torch.Generator().manual_seed(4)
    lens = [100, 70, 200]
    kc, vc, indptr, order, slots = sequences(gen, lens, 16, hkv, d, BF16)
    q = torch.randn(new * 3, hq, d, generator=gen).to(BF16).cuda()
    scale = 1 / math.sqrt(d)
    order = order.clone()
    order[indptr[1] + 2] = kc.shape[0] + 5
    order[indptr[2] + 1] = -7
    said = [100, 70, 10 ** 6]
    held = [100, 70, 16 * 13]

    def ints(x):
        return torch.tensor(x).int().cuda()

    prefix = [h - new for h in held]
    if new == 1:
        out = K.paged_decode_attention_q4(q, kc, vc, indptr.cuda(), order.cuda(), ints(said), scale)
    else:
        out = K.paged_prefill_attention_q4(q, kc, vc, ints([0, new, 2 * new, 3 * new]), indptr.cuda(), order.cuda(), ints(said),
                                           ints(prefix), scale, new, sliding_window_size=window)
    assert K.device_status() == 2
    parts = []
    for b in range(3):
        pages = order[indptr[b]:indptr[b + 1]].long()
        ids = torch.where((pages >= 0) & (pages < kc.shape[0]), pages * 16, torch.full_like(pages, -10 ** 6))
        at = (ids[:, None] + torch.arange(16)).flatten()[:held[b]]
        seen = mask_of(prefix[b], new, False, window if new > 1 else 0)
        parts.append(Q.attention(q[b * new:(b + 1) * new].cpu(), kc, vc, at, seen, scale))
    assert_within(out, *(torch.cat(x) for x in zip(*parts)), BF16)


@pytest.mark.gpu
def test_garbage_behind_a_sequence_and_zero_length():
    """Rows behind the last token, pages that nobody owns and a whole foreign pool's bytes do not reach a result; a row that no
    key is visible to gives zeros."""
    gen = torch.Generator().manual_seed(6)
    lens = [33, 0, 5]
    kc, vc, indptr, order, slots = sequences(gen, lens, 16, 2, 128, F16)
    dirty = [torch.full_like(kc, math.nan), torch.full_like(vc, math.inf)]
    for clean, bad in zip((kc, vc), dirty):     # the sequences' rows, byte by byte
        a, b = clean.view(torch.uint8), bad.view(torch.uint8)
        for s in slots:
            for slot in s.tolist():
                r = slot % 16
                for lo, n in ((64 * r, 64), (1024 + 8 * r, 8)):
                    b[slot // 16, :, lo:lo + n] = a[slot // 16, :, lo:lo + n]
    q = torch.randn(3, 8, 128, generator=gen).to(F16).cuda()
    lens_t = torch.tensor(lens).int().cuda()
    one = K.paged_decode_attention_q4(q, kc, vc, indptr.cuda(), order.cuda(), lens_t, 0.1)
    two = K.paged_decode_attention_q4(q, *dirty, indptr.cuda(), order.cuda(), lens_t, 0.1)
    assert torch.equal(one, two) and (one[1] == 0).all() and torch.isfinite(one).all()
    for new in (2, 70):       # few columns, and the tensor-core tiles
        qo = torch.tensor([0, new, new, 2 * new]).int().cuda()
        q = torch.randn(2 * new, 8, 128, generator=gen).to(F16).cuda()
        prefix = torch.tensor([33 - new, 0, 5 - new]).int().cuda()      # (a block that begins in front of position 0)
        for kw in ({}, dict(sliding_window_size=3), dict(is_cross_attention=True)):
            a, b = (K.paged_prefill_attention_q4(q, *kv, qo, indptr.cuda(), order.cuda(), lens_t, prefix, 0.1, new, **kw)
                    for kv in ((kc, vc), dirty))
            assert torch.equal(a, b) and torch.isfinite(a).all()
            if not kw:
                empty = torch.cat([torch.arange(new) + 33 - new < 0, torch.arange(new) + 5 - new < 0])
                assert (a.cpu()[empty] == 0).all() and (a.cpu()[~empty] != 0).any()
    assert K.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size", [(BF16, 1e-12), (BF16, 1e-4), (BF16, 300.0), (F16, 1e-4), (F16, 300.0)])
def test_sizes_of_keys_values_and_queries(dtype, size):
    """Values and queries far from 1, with scores of order 1."""
    gen = torch.Generator().manual_seed(7)
    lens, hq, hkv, d = [300, 20], 8, 2, 128
    kc, vc, indptr, order, slots = sequences(gen, lens, 16, hkv, d, dtype)
    every = torch.arange(kc.shape[0] * 16).int().cuda()
    v = (torch.randn(len(every), hkv, d, generator=gen) * size).to(dtype)
    K.store_kv_cache_q4(kc, vc, every, torch.randn(len(every), hkv, d, generator=gen).to(dtype).cuda(), v.cuda())
    q = (torch.randn(2, hq, d, generator=gen) * size).to(dtype)
    scale = 0.09 / size
    out = K.paged_decode_attention_q4(q.cuda(), kc, vc, indptr.cuda(), order.cuda(), torch.tensor(lens).int().cuda(), scale)
    parts = [Q.attention(q[b:b + 1], kc, vc, s, torch.ones(1, len(s), dtype=torch.bool), scale) for b, s in enumerate(slots)]
    ref, weighted, _ = (torch.cat(x) for x in zip(*parts))
    err = (out.double().cpu() - ref).abs()
    # as assert_within, with its absolute term in proportion, and a unit of a subnormal f16 output
    assert (err <= 1e-2 * weighted + 2.0 ** -25 * (dtype == F16)).all()
    assert float((out.double().cpu() - ref).norm() / ref.norm()) <= 2 * half_unit(dtype) + (2e-3 if size < 1e-3 and dtype == F16 else 0)


@pytest.mark.gpu
def test_negative_and_zero_scores_scale():
    gen = torch.Generator().manual_seed(8)
    kc, vc, indptr, order, slots = sequences(gen, [90], 16, 2, 128, BF16)
    lens = torch.tensor([90]).int().cuda()
    for new in (1, 3, 100):
        q = torch.randn(new, 16, 128, generator=gen).to(BF16)
        for scale in (-0.09, 0.0):
            prefix = 90 - new
            seen = mask_of(max(prefix, 0), min(new, 90), False, 0)
            if new == 1:
                out = K.paged_decode_attention_q4(q.cuda(), kc, vc, indptr.cuda(), order.cuda(), lens, scale)
                parts = Q.attention(q, kc, vc, slots[0], seen, scale)
            else:
                n = min(new, 90)
                out = K.paged_prefill_attention_q4(q[:n].contiguous().cuda(), kc, vc, torch.tensor([0, n]).int().cuda(),
                                                   indptr.cuda(), order.cuda(), lens, torch.tensor([90 - n]).int().cuda(), scale, n)
                parts = Q.attention(q[:n], kc, vc, slots[0], mask_of(90 - n, n, False, 0), scale)
            assert_within(out, *parts, BF16)


class Layers:
    """A stack of layers over one 4-bit pool and its allocator, with a float64 account of what the pool stands for."""

    def __init__(self, hq, hkv, d, dtype, page_size, requests, longest, layers=2):
        self.gen = torch.Generator().manual_seed(hq + d)
        self.hq, self.hkv, self.d, self.dtype, self.layers = hq, hkv, d, dtype, layers
        pages = requests * -(-longest // page_size) + 3
        self.pool = MHAKVCacheQ4(hkv, layers, d, pages * page_size, dtype)
        self.alloc = CacheManager("cuda", pages, type="naive", page_size=page_size)
        self.table = torch.zeros(requests, longest, dtype=torch.int32, device="cuda")
        self.backend = AttnBackend(SimpleNamespace(head_dim=d, num_kv_heads=hkv), self.pool, self.table, page_size=page_size)
        self.weights = [(1 + 0.2 * torch.randn(d, generator=self.gen)).to(dtype) for _ in range(2)]

    def step(self, reqs, phase, projections):
        """One step of every layer; checks each layer's output against the pool as the layer left it."""
        out_loc = []
        for r in reqs:
            last = int(self.table[r.table_idx, r.cached_len - 1]) if r.cached_len else None
            slots = self.alloc.allocate(r.extend_len, start=r.cached_len, last_slot=last)
            self.table[r.table_idx, r.cached_len:r.device_len] = slots
            out_loc.append(slots)
        batch = Batch(reqs, phase, out_loc=torch.cat(out_loc))
        batch.attn_metadata = (self.backend.build_decode_metadata(reqs) if phase == BatchPhase.DECODE
                               else self.backend.build_prefill_metadata(reqs))
        n = len(batch.out_loc)
        pos = torch.cat([torch.arange(r.cached_len, r.device_len) for r in reqs])
        for layer in range(self.layers):
            qkv = rows(self.gen, n, self.hq + 2 * self.hkv, self.d, self.dtype)
            q, k, v = qkv.cuda().split((self.hq, self.hkv, self.hkv), 1)
            if projections:
                out = self.backend.forward_from_projections(q, k, v, layer, batch, q_norm_weight=self.weights[0].cuda(),
                                                            k_norm_weight=self.weights[1].cuda(), rope_base=1e6)
                ref_q, _ = norm_rotate(q.cpu(), self.weights[0], pos, self.d, 1e-6, 1e6)
                ref_q = ref_q.to(self.dtype)
            else:
                out = self.backend.forward(q.contiguous(), k, v, layer, batch)
                ref_q = q.cpu()
                back = self.pool.load_kv(batch.out_loc, layer)
                assert torch.equal(back[0].cpu(), Q.read(self.pool.k_cache(layer), batch.out_loc).to(self.dtype))
            parts, a = [], 0
            for r in reqs:
                slots = self.table[r.table_idx, :r.device_len].cpu()
                parts.append(Q.attention(ref_q[a:a + r.extend_len], self.pool.k_cache(layer), self.pool.v_cache(layer), slots,
                                         mask_of(r.cached_len, r.extend_len, False, 0), 1 / math.sqrt(self.d)))
                a += r.extend_len
            ref, weighted, size = (torch.cat(x) for x in zip(*parts))
            # (with projections, an element of q can fall a unit of the type off: that times the scores' sizes, as for a rounded key)
            if projections:
                tol = (2 * (size[..., None] * 3 * half_unit(self.dtype)).expm1() + half_unit(self.dtype)) * weighted
                assert ((out.double().cpu() - ref).abs() <= tol + 1e-6).all()
                assert float((out.double().cpu() - ref).norm() / ref.norm()) <= 2 * half_unit(self.dtype)
            else:
                assert_within(out, ref, weighted, size, self.dtype)
        for r in reqs:
            r.complete_one()


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,dtype,page_size", [(16, 4, 128, BF16, 16), (16, 2, 256, F16, 32)])
@pytest.mark.parametrize("projections", [False, True])
def test_engine_steps(hq, hkv, d, dtype, page_size, projections):
    """Prompts, decode steps, a second chunk and a block of a few tokens over one pool, as an engine runs them."""
    engine = Layers(hq, hkv, d, dtype, page_size, 3, 400)
    reqs = [Req(i, 0, n) for i, n in enumerate((150, 17, 64))]
    engine.step(reqs, BatchPhase.PREFILL, projections)
    for _ in range(3):
        engine.step(reqs, BatchPhase.DECODE, projections)
    for r, n in zip(reqs, (30, 3, 100)):
        r.device_len = r.cached_len + n
    engine.step(reqs, BatchPhase.PREFILL, projections)
    for r in reqs:
        r.device_len = r.cached_len + 4
    engine.step(reqs, BatchPhase.TARGET_VERIFY, projections)
    engine.step(reqs, BatchPhase.DECODE, projections)
    assert K.device_status() == 0


def _call(kind, gen, lens, hq=16, hkv=4, d=128, dtype=BF16, new=1):
    kc, vc, indptr, order, slots = sequences(gen, lens, 16, hkv, d, dtype)
    q = torch.randn(len(lens) * new, hq, d, generator=gen).to(dtype).cuda()
    t = [x.cuda() for x in (indptr, order, torch.tensor(lens).int())]
    if kind == "decode":
        return q, lambda **kw: K.paged_decode_attention_q4(q, kc, vc, *t, 0.09, **kw)
    qo = torch.arange(0, len(lens) * new + 1, new).int().cuda()
    prefix = torch.tensor([x - new for x in lens]).int().cuda()
    return q, lambda **kw: K.paged_prefill_attention_q4(q, kc, vc, qo, *t, prefix, 0.09, new, **kw)


KINDS = [("decode", [3000, 40, 700], 1), ("prefill", [3000, 40, 700], 3), ("prefill", [3000, 400, 700], 37),
         ("prefill", [6000], 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,lens,new", KINDS)
def test_streams_graphs_and_two_calls_at_once(kind, lens, new):
    gen = torch.Generator().manual_seed(11)
    q, f = _call(kind, gen, lens, hq=32, hkv=4, new=new)
    q2, g = _call(kind, gen, [x + 5 for x in lens], hq=32, hkv=4, new=new)
    want, want2 = f(), g()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    # two streams at once, and a stream by argument
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = f()
        b = g(stream=s2)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want2)
    # two graphs of one stream, replayed in turn and on new contents
    graphs, outs = [], []
    for call in (f, g):
        with torch.cuda.stream(s1):
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s1):
            outs.append(call())
        graphs.append(graph)
    old = q.clone()
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)
    q.copy_(torch.randn(q.shape, generator=gen).to(q.dtype))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], f())
    q.copy_(old)
    assert torch.equal(f(), want) and K.device_status() == 0


@pytest.mark.gpu
def test_append_and_read_in_a_graph_and_on_a_stream():
    gen = torch.Generator().manual_seed(12)
    kc, vc = (torch.zeros(K.kv_cache_q4_shape(64, 2, 128), dtype=BF16, device="cuda") for _ in range(2))
    qkv = rows(gen, 9, 8, 128, BF16).cuda()
    q, k, v = qkv.split((4, 2, 2), 1)
    slots = torch.randperm(64, generator=gen)[:9].int().cuda()
    pos = torch.arange(9).int().cuda()

    def step():
        r = K.qk_norm_rope_store_q4(q, k, v, None, None, pos, slots, kc, vc, rope_base=1e4)
        return r, *K.load_kv_cache_q4(kc, vc, slots)

    want = [x.clone() for x in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = step()
    kc.zero_()
    vc.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    K.store_kv_cache_q4(kc, vc, slots, k.contiguous(), v, stream=s)
    s.synchronize()
    assert torch.equal(Q.read(kc, slots).float(), Q.values(*Q.quantise(k.cpu())).float())


@pytest.mark.gpu
def test_many_short_sequences_and_offsets_beyond_32_bits():
    """Two thousand sequences (more counters than a workspace's header has, with eight heads), and a pool of more than 2^32 bytes."""
    gen = torch.Generator().manual_seed(13)
    lens = [1 + i % 37 for i in range(2100)]
    kc, vc, indptr, order, slots = sequences(gen, lens, 16, 8, 128, BF16)
    q = torch.randn(len(lens), 16, 128, generator=gen).to(BF16)
    out = K.paged_decode_attention_q4(q.cuda(), kc, vc, indptr.cuda(), order.cuda(), torch.tensor(lens).int().cuda(), 0.09)
    for b in (0, 1, 35, 36, 37, 1000, 2099):
        parts = Q.attention(q[b:b + 1], kc, vc, slots[b], torch.ones(1, lens[b], dtype=torch.bool), 0.09)
        assert_within(out[b:b + 1], *parts, BF16)
    del kc, vc
    blocks = (1 << 32) // (8 * 1152) + 100
    kc, vc = (torch.zeros(blocks, 8, 576, dtype=BF16, device="cuda") for _ in range(2))
    n = 50
    at = torch.arange(n).int() + 16 * (blocks - 40)
    k, v = rows(gen, n, 8, 128, BF16), rows(gen, n, 8, 128, BF16)
    K.store_kv_cache_q4(kc, vc, at.cuda(), k.cuda(), v.cuda())
    back = K.load_kv_cache_q4(kc, vc, at.cuda())
    assert torch.equal(back[0].cpu(), Q.values(*Q.quantise(k)).to(BF16)) and torch.equal(back[1].cpu(), Q.values(*Q.quantise(v)).to(BF16))
    pages = torch.arange(blocks - 40, blocks - 36).int().cuda()
    small = [Q_pool[blocks - 40:].cpu() for Q_pool in (kc, vc)]
    for new in (1, 2, 30):
        q = torch.randn(new, 16, 128, generator=gen).to(BF16)
        args = (torch.tensor([0, 4]).int().cuda(), pages, torch.tensor([n]).int().cuda())
        if new == 1:
            out = K.paged_decode_attention_q4(q.cuda(), kc, vc, *args, 0.09)
        else:
            out = K.paged_prefill_attention_q4(q.cuda(), kc, vc, torch.tensor([0, new]).int().cuda(), *args,
                                               torch.tensor([n - new]).int().cuda(), 0.09, new)
        assert_within(out, *Q.attention(q, *small, torch.arange(n), mask_of(n - new, new, False, 0), 0.09), BF16)
    assert K.device_status() == 0


@pytest.mark.gpu
def test_a_long_prefill_without_memory_for_its_pages(monkeypatch):
    gen = torch.Generator().manual_seed(14)
    _, f = _call("prefill", gen, [6000], hq=32, hkv=4, new=2048)
    want = f()
    _lib.host.set_pages_maker(lambda nbytes, index, stream: None)
    try:
        got = f()
    finally:
        _lib.host.set_pages_maker(K._make_pages)
    # two forms, each within half a unit of the output and its operands' roundings of the other
    assert float((got.double() - want.double()).norm() / want.double().norm()) <= 2 * half_unit(BF16)


@pytest.mark.gpu
def test_row_pointers_that_fit_no_batch():
    """Page pointers that lay more blocks end to end than any batch holds are reported and nothing is read; query pointers beyond
    the rows of q end with them."""
    gen = torch.Generator().manual_seed(12)
    q, decode = _call("decode", gen, [300, 17])
    before = decode()
    batch, pages = 16384, 4096
    kc = torch.zeros(K.kv_cache_q4_shape(4096, 1, 128), dtype=BF16, device="cuda")
    ends = torch.tensor([0, pages] * (batch // 2) + [0]).int().cuda()
    ids = torch.zeros(pages, dtype=torch.int32, device="cuda")
    K.paged_decode_attention_q4(torch.ones(batch, 1, 128, dtype=BF16, device="cuda"), kc, kc, ends, ids,
                                torch.full((batch,), 1 << 20, dtype=torch.int32, device="cuda"), 0.1, page_size=256)
    assert K.device_status() == 2
    assert torch.equal(decode(), before) and K.device_status() == 0

    kc, vc, indptr, order, _ = sequences(gen, [50, 40], 16, 4, 128, BF16)
    q = torch.randn(5, 16, 128, generator=gen).to(BF16).cuda()

    def attend(qo):
        return K.paged_prefill_attention_q4(q, kc, vc, torch.tensor(qo).int().cuda(), indptr.cuda(), order.cuda(),
                                            torch.tensor([50, 40]).int().cuda(), torch.tensor([47, 38]).int().cuda(), 0.1, 4)

    assert torch.equal(attend([0, 3, 9]), attend([0, 3, 5]))
