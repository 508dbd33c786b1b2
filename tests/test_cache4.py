"""The paged 4-bit cache: refusals on the CPU; append, read, attention and eviction on a B200 against 64 bits."""
import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from ascend_rsfa import _capi
from ascend_rsfa import flash_attention_forward as fa
from ascend_rsfa import kv_cache as kc
from ascend_rsfa import rotary as ro
from oracle import operators_ref as ref

lib = _capi.load()
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
DTYPES = [torch.float16, torch.bfloat16]


def rows(dev, shape, dtype, seed, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * std).to(dtype)


def make(dev, lengths, H, D, page, dtype, seed=0, room=None, std=1.0):
    """A cache in random pages whose slots in use hold N(0, 1) rows and whose other bytes are 0xff: NaN scales."""
    g = torch.Generator(device=dev).manual_seed(seed)
    B, n = len(lengths), -(-max(max(lengths), room or 1) // page)
    spare = 3
    table = torch.randperm(B * n + spare, generator=g, device=dev)[: B * n].to(torch.int32).view(B, n)
    kv = torch.full((B * n + spare, H, page, 5 * D // 4), 255, dtype=torch.uint8, device=dev)
    for b, m in enumerate(lengths):
        if m:
            k, v = ((torch.randn(m, H, D, generator=g, device=dev) * std).to(dtype) for _ in range(2))
            slot = torch.arange(m, device=dev)
            kv[table[b].long()[slot // page], :, slot % page] = ref.records(k.reshape(-1, D), v.reshape(-1, D)).view(m, H, -1)
    return kv, table, torch.tensor(lengths, dtype=torch.int32, device=dev)


def check_attention(got, q, kv, table, lengths, scale, counts=None, lse=None, weight=None, weight_before=None):
    """The operator's own roundings.  A result is sum p s (u - 8) + sum p (m + 8 s): p * s is rounded to fp16, half a step of
    2^-11, and p to the cache's type, half a step of that, so the two sums are off by 2^-11 sum p s |u - 8| and by half a
    step of sum p |m + 8 s|; the result is rounded to 16 bits.  The 32-bit sums sum P (u - 8), sum p m and sum p s are cut off
    at 2^-24 of what they come to, some 2^8 times: 2^-16 of sum p s |u - 8| and sum p (|m| + 8 s), which the difference of the
    last two can be far below.  (That covers P below fp16's normal numbers, an absolute 2^-25 where the largest is 2^10.)
    A score is a sum of D products of at most `terms` in total, rounded a few times in 32 bits, and an exponential with a
    relative error of 2^-22: weights are off by 2^-19 (1 + terms) at most."""
    o, want_lse, weights, (parts, middles, both, sizes, terms) = ref.attention(q, kv, table, lengths, scale, counts)
    off = 2.0 ** -19 * (1 + terms)
    bound = (HALF_STEP[q.dtype] * (o.abs() + middles) + 2.0 ** -11 * parts + 2 * off[..., None] * sizes + 2.0 ** -16 * (parts + both)
             + TINY[q.dtype])
    err = (got.double() - o).abs()
    assert bool((err <= bound).all()), (float(err.max()), float((err - bound).max()))
    if lse is not None:
        seen = want_lse > -math.inf
        assert bool((lse[~seen] == -math.inf).all())
        assert bool(((lse.double() - want_lse).abs()[seen] <= (off + 2.0 ** -22 * want_lse.abs())[seen] + 2.0 ** -20).all())
    if weight is not None:
        P, B, H = kv.shape[2], q.shape[0], kv.shape[1]
        want = weight_before.double().clone()
        for b in range(B):
            n = int(lengths[b])
            slot = torch.arange(n, device=q.device)
            for h in range(H):
                want[table[b].long()[slot // P], h, slot % P] += weights[b, h]
        rel = 2.0 * float(off.max()) + 2.0 ** -20
        # the sum of up to eight rows, then half a step of 2^-24 for every block of rows that is added, and one for `want`
        blocks = -(-q.shape[1] // H * q.shape[2] // 8) + 1
        assert bool(((weight.double() - want).abs() <= rel * (want - weight_before.double()) + 2.0 ** -24 * blocks * want.abs() + 1e-30).all())


# ------------------------------------------------------------------ without a GPU

def test_refusals_need_no_device():
    kv = torch.zeros(4, 2, 16, 80, dtype=torch.uint8)
    q = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    table, lengths = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kc.cache4_attention(q, kv, table, lengths, 0.125)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kc.cache4_append(q, q, kv, table, lengths)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kc.cache4_read(kv, table, lengths, 4, torch.float16)
    for args in ((4, 2, 16, 32), (4, 2, 24, 64), (4, 2, 8, 64), (0, 2, 16, 64), (4, 0, 16, 64), (4, 2, 2048, 64)):
        with pytest.raises(ValueError):
            kc.cache4_empty(*args, device="cpu")
    for budget, recent in ((0, 0), (4, 5), (4, -1)):
        with pytest.raises(ValueError):
            kc.cache4_evict(kv, None, None, table, lengths, budget, recent)
    with pytest.raises(ValueError, match="weight and position"):
        kc.cache4_evict(kv, None, None, table, lengths, 4)
    kv, weight, position = kc.cache4_empty(4, 2, 16, 64, device="cpu")
    assert kv.shape == (4, 2, 16, 80) and weight.shape == position.shape == (4, 2, 16)


def c_cache(**kw):
    base = dict(kv=4096, weight=4096, position=4096, table=4096, lengths=4096, kv_stride=(2 * 16 * 80, 16 * 80), weight_stride=(32, 16),
                position_stride=(32, 16), table_stride=4, batch=2, heads=2, head_dim=64, page_size=16, pages=4, max_pages=4, dtype=0)
    c = _capi.Cache4()
    for name, value in {**base, **kw}.items():
        setattr(c, name, (ctypes.c_int64 * 2)(*value) if isinstance(value, tuple) else value)
    return ctypes.byref(c)


def test_c_refusals_need_no_device():
    bad, p = _capi.RSFA_ERR_INVALID_ARGUMENT, ctypes.c_void_p(4096)
    st = (ctypes.c_int64 * 8)(*([512, 256, 64, 1] * 2))
    broken = [dict(kv=None), dict(table=None), dict(lengths=None), dict(kv=4104), dict(batch=0), dict(heads=0), dict(pages=0), dict(max_pages=0),
              dict(head_dim=48), dict(page_size=24), dict(page_size=8), dict(page_size=2048), dict(dtype=2), dict(kv_stride=(2560, 1272)),
              dict(kv_stride=(1280, 640)), dict(weight_stride=(8, 16)), dict(position_stride=(32, 8)), dict(table_stride=-4)]
    for kw in broken:
        c = c_cache(**kw)
        assert lib.rsfa_cache4_append(c, p, p, 4, st, None, p, st, None) == bad, kw
        assert lib.rsfa_cache4_read(c, p, p, 4, st, None, None) == bad, kw
        assert lib.rsfa_cache4_attention(c, p, p, p, 2, 4, st, None, 0.5, p, 1 << 40, None) == bad, kw
        assert lib.rsfa_cache4_evict(c, 8, 2, p, p, 1 << 40, None) == bad, kw
    assert lib.rsfa_cache4_read(c_cache(head_dim=32), p, p, 4, st, None, None) == _capi.RSFA_ERR_UNSUPPORTED
    assert lib.rsfa_cache4_read(c_cache(max_pages=1 << 28), p, p, 4, st, None, None) == _capi.RSFA_ERR_TOO_LARGE
    c, odd = c_cache(), (ctypes.c_int64 * 8)(*([512, 256, 60, 1] * 2))
    assert lib.rsfa_cache4_append(c, None, p, 4, st, None, p, st, None) == bad
    assert lib.rsfa_cache4_append(c, p, p, 0, st, None, p, st, None) == bad
    assert lib.rsfa_cache4_append(c, p, p, 4, odd, None, p, st, None) == bad
    assert lib.rsfa_cache4_append(c, p, p, 4, st, None, None, None, None) == bad              # position without positions
    assert lib.rsfa_cache4_append(c_cache(position=None), p, p, 4, st, None, p, st, None) == bad
    assert lib.rsfa_cache4_attention(c, p, p, None, 2, 4, st, None, 0.5, p, 1 << 40, None) == bad   # weights need the lse
    assert lib.rsfa_cache4_attention(c, p, p, p, 3, 4, st, None, 0.5, p, 1 << 40, None) == bad
    assert lib.rsfa_cache4_attention(c, p, p, p, 2, 4, st, None, float("nan"), p, 1 << 40, None) == bad
    assert lib.rsfa_cache4_evict(c, 0, 0, p, p, 1 << 40, None) == bad
    assert lib.rsfa_cache4_evict(c, 8, 9, p, p, 1 << 40, None) == bad
    assert lib.rsfa_cache4_evict(c, 8, 2, ctypes.c_void_p(8192), p, 16, None) == bad            # scratch too small
    assert lib.rsfa_cache4_evict(c, 8, 2, p, p, 1 << 40, None) == bad                           # new_lengths are lengths
    assert lib.rsfa_cache4_evict(c_cache(weight=None), 8, 2, ctypes.c_void_p(8192), p, 1 << 40, None) == bad
    assert lib.rsfa_cache4_evict_workspace(2, 2, 8) > 0 and lib.rsfa_cache4_evict_workspace(0, 2, 8) == bad
    assert lib.rsfa_cache4_attention_workspace(c_cache(head_dim=48), 2, 1) == bad and lib.rsfa_cache4_attention_workspace(c, 3, 1) == bad


def test_more_tiles_than_are_counted_are_refused():
    # 2^20 sequences of up to 2^30 slots that share their pages: 2^25 tiles of each of 2 heads
    p, st = ctypes.c_void_p(4096), (ctypes.c_int64 * 8)(*([512, 256, 64, 1] * 2))
    c = c_cache(batch=1 << 20, max_pages=1 << 26, table_stride=0, weight=None)
    assert lib.rsfa_cache4_attention(c, p, p, p, 2, 4, st, None, 0.5, p, 1 << 62, None) == _capi.RSFA_ERR_TOO_LARGE


def test_oracle_record_round_trip():
    for dtype in DTYPES:
        for D in (64, 128, 256):
            x, y = (torch.randn(9, D, generator=torch.Generator().manual_seed(s)).to(dtype) for s in (1, 2))
            k, v, _ = ref.values(ref.records(x, y), dtype)
            for a, b in ((x, k), (y, v)):
                f = a.double().view(9, -1, 32)
                step = (f.max(-1).values - f.min(-1).values)[..., None] / 15
                # half a step, and at the top 15 steps that are a rounding short
                assert bool(((f - b.view_as(f)).abs() <= step * (0.5 + 16 * HALF_STEP[dtype])).all())


# ------------------------------------------------------------------ append and read

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,page,held,S", [(64, 1, 16, [0], 1), (64, 3, 32, [5, 0, 31], 7), (128, 2, 16, [15, 1], 33), (128, 8, 64, [100, 63, 0, 7], 1),
                                             (256, 2, 128, [0, 130], 19), (256, 1, 1024, [3], 2)])
def test_append_writes_the_records_and_nothing_else(cuda_device, dtype, D, H, page, held, S):
    B = len(held)
    kv, table, _ = make(cuda_device, held, H, D, page, dtype, room=max(held) + S)
    weight, position = torch.full(kv.shape[:3], 7.0, device=cuda_device), torch.full(kv.shape[:3], -5, dtype=torch.int32, device=cuda_device)
    lengths = torch.tensor([n + S for n in held], dtype=torch.int32, device=cuda_device)
    k, v = rows(cuda_device, (B, S, H, D), dtype, 1).transpose(1, 2), rows(cuda_device, (B, H, S, D), dtype, 2, 3.0)
    v[0, 0, 0, :32] = 0.25                                        # a group without a range
    positions = torch.arange(B * S, device=cuda_device, dtype=torch.int32).view(B, S) + 1000
    want, want_w, want_p = kv.clone(), weight.clone(), position.clone()
    for b in range(B):
        slot = torch.arange(held[b], held[b] + S, device=cuda_device)
        at = (table[b].long()[slot // page], slice(None), slot % page)
        want[at] = ref.records(k[b].transpose(0, 1).reshape(-1, D), v[b].transpose(0, 1).reshape(-1, D)).view(S, H, -1)
        want_w[at], want_p[at] = 0.0, positions[b][:, None]
    kc.cache4_append(k, v, kv, table, lengths, weight=weight, position=position, positions=positions)
    assert torch.equal(kv, want) and torch.equal(weight, want_w) and torch.equal(position, want_p)
    n = int(lengths.max()) + 3
    starts = torch.tensor([b - 1 for b in range(B)], dtype=torch.int32, device=cuda_device)
    for st in (None, starts):
        rk, rv = kc.cache4_read(kv, table, lengths, n, dtype, starts=st)
        for b in range(B):
            first = 0 if st is None else int(st[b])
            for h in range(H):
                kk, vv, _ = ref.values(ref.rows_of(kv, table, b, h, int(lengths[b])), dtype)
                for got, val in ((rk[b, h], kk), (rv[b, h], vv)):
                    exp = torch.zeros(n, D, dtype=torch.float64, device=cuda_device)
                    lo, hi = max(first, 0), min(first + n, int(lengths[b]))
                    exp[lo - first:hi - first] = val[lo:hi]
                    # one rounding to 16 bits and one to 32 of s u + m
                    assert bool(((got.double() - exp).abs() <= (HALF_STEP[dtype] + 2.0 ** -23) * exp.abs() + 2.0 ** -23 * val.abs().max() + TINY[dtype]).all())
    fa.device_status()


@pytest.mark.gpu
def test_append_of_padded_rows_and_sequences_not_in_use(cuda_device):
    held, S, H, D, page = [3, 0, 10, 20], 6, 2, 64, 16
    kv, table, _ = make(cuda_device, held, H, D, page, torch.float16, room=32)
    counts = torch.tensor([6, 0, 2, 4], dtype=torch.int32, device=cuda_device)
    lengths = torch.tensor([9, 0, 12, 24], dtype=torch.int32, device=cuda_device)
    k, v = rows(cuda_device, (4, H, S, D), torch.float16, 1), rows(cuda_device, (4, H, S, D), torch.float16, 2)
    k[0, 1, 0, 3], v[2, 0, 1, 40] = math.inf, math.nan
    k[1], v[1] = math.nan, math.nan                                # padding
    want = kv.clone()
    for b in range(4):
        c = int(counts[b])
        slot = torch.arange(held[b], held[b] + c, device=cuda_device)
        want[table[b].long()[slot // page], :, slot % page] = ref.records(k[b, :, :c].transpose(0, 1).reshape(-1, D),
                                                                         v[b, :, :c].transpose(0, 1).reshape(-1, D)).view(c, H, 5 * D // 4)
    kc.cache4_append(k, v, kv, table, lengths, counts=counts)
    rk, rv = kc.cache4_read(kv, table, lengths, 24, torch.float16)
    # NaN has many bit patterns: compared as values
    wk, wv = kc.cache4_read(want, table, lengths, 24, torch.float16)
    assert torch.equal(rk.nan_to_num(9.5), wk.nan_to_num(9.5)) and torch.equal(rv.nan_to_num(9.5), wv.nan_to_num(9.5))
    assert bool(rk[0, 1, 3, :32].isnan().all()) and not bool(rk[0, 1, 3, 32:].isnan().any()) and bool(rv[2, 0, 11, 32:].isnan().all())
    assert int(rk.isnan().sum()) == int(rv.isnan().sum()) == 32
    untouched = torch.ones(kv.shape[:3], dtype=torch.bool, device=cuda_device)
    for b in range(4):
        slot = torch.arange(held[b], held[b] + int(counts[b]), device=cuda_device)
        untouched[table[b].long()[slot // page], :, slot % page] = False
    assert torch.equal(kv[untouched], want[untouched])
    # without counts a sequence of length zero takes nothing, one shorter than S its last rows
    lengths = torch.tensor([0, 2, 6, 6], dtype=torch.int32, device=cuda_device)
    kv2 = kv.clone()
    kc.cache4_append(v[[3]].expand(4, -1, -1, -1), v[[3]].expand(4, -1, -1, -1), kv2, table, lengths)
    a, b = kc.cache4_read(kv2, table, lengths, 6, torch.float16)
    assert torch.equal(a[1, :, :2], a[2, :, 4:]) and bool((a[0] == 0).all())
    fa.device_status()


# ------------------------------------------------------------------ attention

SHAPES = [  # Hq, H, S, D, page, lengths
    (1, 1, 1, 64, 16, [1]), (2, 2, 1, 128, 64, [1, 0, 2]), (8, 1, 1, 128, 16, [15, 16, 17, 31, 32, 33]), (8, 8, 1, 64, 32, [500, 1, 77]),
    (32, 8, 1, 128, 64, [1000]), (12, 4, 1, 256, 16, [333, 64]), (16, 1, 1, 128, 128, [700, 129]), (6, 2, 3, 64, 16, [2, 3, 100, 0]),
    (20, 2, 1, 64, 32, [257, 40]), (4, 4, 5, 128, 64, [5, 64, 65, 900]), (4, 1, 9, 256, 32, [9, 200]), (48, 2, 1, 128, 16, [97]),
    (2, 1, 40, 64, 16, [40, 123]), (1, 1, 1, 256, 1024, [2500]), (3, 3, 1, 128, 64, [64, 32, 96, 16, 48, 80, 112] * 6),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention(cuda_device, dtype, shape):
    Hq, H, S, D, page, lengths = shape
    B = len(lengths)
    kv, table, n = make(cuda_device, lengths, H, D, page, dtype, seed=Hq + D)
    q = rows(cuda_device, (B, S, Hq, D), dtype, 5, 2.0).transpose(1, 2)
    scale = 1 / math.sqrt(D)
    before = torch.rand(kv.shape[:3], device=cuda_device)
    weight = before.clone()
    kv0 = kv.clone()
    o, lse = kc.cache4_attention(q, kv, table, n, scale, weight=weight, want_lse=True)
    assert o.dtype == dtype and o.shape == q.shape and torch.equal(kv, kv0)
    check_attention(o, q, kv, table, n, scale, None, lse, weight, before)
    assert torch.equal(kc.cache4_attention(q.contiguous(), kv, table, n, scale), o)
    if S > 1:
        counts = torch.tensor([(2 * b + 1) % (S + 1) for b in range(B)], dtype=torch.int32, device=cuda_device)
        weight = before.clone()
        o, lse = kc.cache4_attention(q, kv, table, n, scale, counts=counts, weight=weight, want_lse=True)
        check_attention(o, q, kv, table, n, scale, counts, lse, weight, before)
    fa.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,Hq,H", [(64, 4, 4), (128, 8, 2), (128, 16, 1), (256, 3, 1)])
def test_attention_of_wide_scores_and_scales(cuda_device, dtype, D, Hq, H):
    """Scores that rise along the sequence (the reference is raised again and again), near one-hot rows, negative
    and zero scales, and V rows whose sizes differ by many powers of two."""
    n = 600
    kv, table, lengths = make(cuda_device, [n], H, D, 32, dtype, seed=1, room=n)
    k, v = rows(cuda_device, (1, H, n, D), dtype, 3), rows(cuda_device, (1, H, n, D), dtype, 4)
    ramp = torch.linspace(0.02, 4, n, device=cuda_device)
    kc.cache4_append((k.float() * ramp[:, None]).to(dtype), (v.float() * 2.0 ** torch.linspace(-9, 9, n, device=cuda_device)[:, None]).to(dtype),
                     kv, table, lengths)
    q = rows(cuda_device, (1, Hq, 1, D), dtype, 6, 2.0)
    for scale in (1 / math.sqrt(D), 1.0, -0.1, 0.0):
        o, lse = kc.cache4_attention(q, kv, table, lengths, scale, want_lse=True)
        check_attention(o, q, kv, table, lengths, scale, None, lse)
    for size in (2.0 ** -12, 2.0 ** 8):                             # q of other sizes than one
        qs = (q.float() * size).to(dtype)
        check_attention(kc.cache4_attention(qs, kv, table, lengths, 0.1 / size), qs, kv, table, lengths, 0.1 / size)
    kv.zero_()                                                      # scales and minima of zero
    o, lse = kc.cache4_attention(q, kv, table, lengths, 1.0, want_lse=True)
    assert bool((o == 0).all()) and torch.allclose(lse, torch.full_like(lse, math.log(n)), atol=1e-5)


@pytest.mark.gpu
def test_attention_leaves_nan_where_it_is_and_ignores_what_is_not_in_use(cuda_device):
    dtype, H, D = torch.bfloat16, 2, 128
    kv, table, lengths = make(cuda_device, [40, 70, 0], H, D, 16, dtype, room=80)       # bytes not in use are NaN already
    table = torch.cat((table, torch.full((3, 2), -1, dtype=torch.int32, device=cuda_device)), 1)
    table[0, 3:], table[2] = 2 ** 30, -7                                                 # pages that no length reaches
    q = rows(cuda_device, (3, 4, 1, D), dtype, 1)
    o, lse = kc.cache4_attention(q, kv, table, lengths, 0.1, want_lse=True)
    assert bool(torch.isfinite(o).all()) and bool((o[2] == 0).all()) and bool((lse[2] == -math.inf).all())
    check_attention(o, q, kv, table, lengths, 0.1, None, lse)
    k = rows(cuda_device, (3, H, 1, D), dtype, 2)
    k[0, 1] = math.nan
    kc.cache4_append(k, k, kv, table, lengths)
    o2 = kc.cache4_attention(q, kv, table, lengths, 0.1)
    assert bool(o2[0, 2:].isnan().all()) and bool(torch.isfinite(o2[0, :2]).all()) and bool(torch.isfinite(o2[1:]).all())
    qn = q.clone()
    qn[1, 3, 0, 5] = math.nan
    o3 = kc.cache4_attention(qn, kv, table, lengths, 0.1)
    assert bool(o3[1, 3].isnan().all()) and torch.equal(o3[1, :3], o2[1, :3])
    fa.device_status()


@pytest.mark.gpu
def test_bad_pages_and_lengths_are_reported_and_nothing_outside_is_touched(cuda_device):
    dtype, H, D, page = torch.float16, 2, 64, 16
    kv, table, lengths = make(cuda_device, [40, 30], H, D, page, dtype, room=48)
    weight, position = torch.rand(kv.shape[:3], device=cuda_device), torch.zeros(kv.shape[:3], dtype=torch.int32, device=cuda_device)
    q, k = rows(cuda_device, (2, 4, 1, D), dtype, 1), rows(cuda_device, (2, H, 1, D), dtype, 2)
    positions = torch.ones(2, 1, dtype=torch.int32, device=cuda_device)
    fa.device_status()

    def calls(table, lengths):
        kc.cache4_append(k, k, kv, table, lengths, weight=weight, position=position, positions=positions)
        yield
        kc.cache4_read(kv, table, lengths, 48, dtype)
        yield
        o = kc.cache4_attention(q, kv, table, lengths, 0.125)
        assert bool(torch.isfinite(o[0]).all())
        yield
        kc.cache4_attention(q, kv, table, lengths, 0.125, weight=weight)
        yield
        kc.cache4_evict(kv, weight, position, table, lengths, 8, 2)
        yield

    for page_number in (-1, kv.shape[0], 2 ** 31 - 1):
        bad = table.clone()
        bad[1, 1] = page_number
        for _ in calls(bad, lengths):
            with pytest.raises(RuntimeError, match="device status 0x20002"):
                fa.device_status()
    for length in (-3, 49, 2 ** 31 - 1):
        bad = lengths.clone()
        bad[1] = length
        for _ in calls(table, bad):
            with pytest.raises(RuntimeError, match="device status 0x20003"):
                fa.device_status()
    # the library goes on
    o = kc.cache4_attention(q, kv, table, torch.tensor([8, 8], dtype=torch.int32, device=cuda_device), 0.125)
    assert bool(torch.isfinite(o).all())
    fa.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("H,D,lengths", [(8, 128, [30000]), (1, 64, [70001, 3]), (2, 256, [9000, 0, 5000])])
def test_attention_over_long_sequences(cuda_device, H, D, lengths):
    kv, table, n = make(cuda_device, lengths, H, D, 128, torch.bfloat16, seed=3)
    q = rows(cuda_device, (len(lengths), 2 * H, 1, D), torch.bfloat16, 4, 2.0)
    before = torch.zeros(kv.shape[:3], device=cuda_device)
    weight = before.clone()
    o, lse = kc.cache4_attention(q, kv, table, n, 0.1, weight=weight, want_lse=True)
    check_attention(o, q, kv, table, n, 0.1, None, lse, weight, before)


@pytest.mark.gpu
def test_attention_over_pages_beyond_32_bits(cuda_device):
    """One layer of a cache tensor that all layers share: page strides that put the last pages behind 2^32 bytes."""
    H, D, page, layers = 2, 128, 64, 4000
    every = torch.empty((60, layers, H, page, 160), dtype=torch.uint8, device=cuda_device)
    kv = every[:, 3999]
    small, table, n = make(cuda_device, [3000], H, D, page, torch.float16, room=3000)
    kv[: small.shape[0]].copy_(small)
    table = (59 - table).to(torch.int32)
    kv.copy_(kv.flip(0))
    assert kv.stride(0) * 59 > 2 ** 32
    q = rows(cuda_device, (1, 4, 1, D), torch.float16, 4)
    check_attention(kc.cache4_attention(q, kv, table, n, 0.1), q, kv, table, n, 0.1)
    k = rows(cuda_device, (1, H, 1, D), torch.float16, 5)
    kc.cache4_append(k, k, kv, table, n)
    got = kc.cache4_read(kv, table, n, 1, torch.float16, starts=n - 1)[0]
    assert torch.equal(ref.rows_of(kv, table, 0, 1, 3000)[-1], ref.records(k[0, 1], k[0, 1])[0])
    assert bool(torch.isfinite(got).all())


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,H,S,D", [(4, 4, 1, 64), (16, 2, 1, 128), (16, 1, 1, 128), (3, 1, 2, 256), (8, 1, 5, 64)])
def test_weights_with_a_table_far_wider_than_the_cache(cuda_device, Hq, H, S, D):
    """The scores are not kept then but computed again."""
    lengths = [100, S, 333]
    kv, table, n = make(cuda_device, lengths, H, D, 32, torch.float16, seed=2)
    wide = torch.full((3, 4096), -1, dtype=torch.int32, device=cuda_device)
    wide[:, : table.shape[1]] = table
    q = rows(cuda_device, (3, Hq, S, D), torch.float16, 1, 2.0)
    before = torch.rand(kv.shape[:3], device=cuda_device)
    weight = before.clone()
    o, lse = kc.cache4_attention(q, kv, wide, n, 0.1, weight=weight, want_lse=True)
    check_attention(o, q, kv, wide, n, 0.1, None, lse, weight, before)
    fa.device_status()


@pytest.mark.gpu
def test_pages_and_heads_in_any_order_of_storage(cuda_device):
    dtype, H, D, page = torch.bfloat16, 3, 64, 16
    plain, table, n = make(cuda_device, [50, 17], H, D, page, dtype)
    P = plain.shape[0]
    kv = torch.empty((H, P + 2, page, 80), dtype=torch.uint8, device=cuda_device)[:, 1:P + 1].transpose(0, 1)      # heads outermost, a gap
    weight = torch.empty((H, 2, P, page), device=cuda_device)[:, 1].transpose(0, 1)
    position = torch.empty((P, H, 2 * page), dtype=torch.int32, device=cuda_device)[..., page:]
    kv.copy_(plain), weight.copy_(torch.rand(P, H, page, device=cuda_device)), position.copy_(torch.arange(P * H * page, device=cuda_device).view(P, H, page))
    q, k = rows(cuda_device, (2, 6, 1, D), dtype, 1), rows(cuda_device, (2, H, 1, D), dtype, 2)
    dense = [t.contiguous() for t in (kv, weight, position)]
    pos = torch.tensor([[9000], [9001]], dtype=torch.int32, device=cuda_device)
    table = torch.stack((table, table), -1).flatten(1)[:, ::2].contiguous() if table.shape[1] > 1 else table
    rows_of_table = torch.cat((table, table), 1)[:, : table.shape[1]]                                                # a row stride of its own
    out = []
    for kv_, w_, p_, t_ in ((kv, weight, position, rows_of_table), (*dense, table)):
        kc.cache4_append(k, k, kv_, t_, n, weight=w_, position=p_, positions=pos)
        out.append([kc.cache4_attention(q, kv_, t_, n, 0.1, weight=w_), *kc.cache4_read(kv_, t_, n, 50, dtype), kc.cache4_evict(kv_, w_, p_, t_, n, 20, 3),
                    kv_.contiguous(), w_.contiguous(), p_.contiguous()])
    for a, b in zip(*out):
        assert torch.equal(a, b)
    fa.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dropped", [0, 1, 5])
def test_a_wait_that_runs_out_is_reported(cuda_device, dropped):
    """The loads of every warp's first, second or sixth tile are left out: the kernel returns by itself and says so, and
    the next call is right.  Nothing is in flight for those tiles.  (15000 tiles: at least eight per warp of 148
    multiprocessors with twelve each.)"""
    kv, table, n = make(cuda_device, [60000], 8, 128, 64, torch.float16)
    q = rows(cuda_device, (1, 8, 1, 128), torch.float16, 1)
    want = kc.cache4_attention(q, kv, table, n, 0.1)
    fa.device_status()
    limit = int(lib.rsfa_get_option(b"wait_limit_ms"))
    try:
        fa.set_option("wait_limit_ms", 1)
        fa.set_option("test_drop_load", dropped)
        kc.cache4_attention(q, kv, table, n, 0.1)
        torch.cuda.synchronize()
    finally:
        fa.set_option("test_drop_load", -1)
        fa.set_option("wait_limit_ms", limit)
    with pytest.raises(RuntimeError, match="device status 0x10028"):
        fa.device_status()
    assert torch.equal(kc.cache4_attention(q, kv, table, n, 0.1), want)
    fa.device_status()


@pytest.mark.gpu
def test_check_status_option_makes_the_next_call_fail(cuda_device):
    kv, table, n = make(cuda_device, [20], 1, 64, 16, torch.float16)
    q = rows(cuda_device, (1, 1, 1, 64), torch.float16, 1)
    rope = ro.rotary_table(4, 64, device=cuda_device)
    fa.device_status()
    try:
        fa.set_option("check_status", 1)
        kc.cache4_attention(q, kv, table + 1000, n, 0.1)
        torch.cuda.synchronize()
        for call in (lambda: kc.cache4_attention(q, kv, table, n, 0.1), lambda: ro.rotary(q, None, rope), lambda: kc.cache4_read(kv, table, n, 4, torch.float16)):
            with pytest.raises(RuntimeError, match="device status"):
                call()
        with pytest.raises(RuntimeError, match="0x20002"):
            fa.device_status()
        kc.cache4_attention(q, kv, table, n, 0.1)
    finally:
        fa.set_option("check_status", 0)
    fa.device_status()


# ------------------------------------------------------------------ eviction

@pytest.mark.gpu
@pytest.mark.parametrize("D,H,page,lengths,budget,recent", [
    (64, 2, 16, [40, 10, 0, 33], 32, 4), (128, 1, 64, [1000, 257], 256, 0), (128, 3, 32, [65], 64, 64), (256, 2, 128, [5000, 4097, 130], 129, 100),
    (64, 1, 16, [1, 2, 3], 1, 1), (128, 2, 128, [9000], 7000, 500), (64, 1, 1024, [50000], 4096, 1000),
])
@pytest.mark.parametrize("ties", [False, True])
def test_evict(cuda_device, D, H, page, lengths, budget, recent, ties):
    dtype = torch.float16
    B = len(lengths)
    kv, table, n = make(cuda_device, [min(m, 300) for m in lengths], H, D, page, dtype, room=max(lengths))
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(8)
    kv = torch.randint(0, 256, kv.shape, generator=g, device=cuda_device, dtype=torch.uint8)
    weight = torch.rand(kv.shape[:3], generator=g, device=cuda_device)
    if ties:
        weight = (weight * 4).floor()                              # a handful of values, many zeros
        weight[weight == 3] = math.nan
        weight[weight == 2] = -1.0
    # positions of a cache that has been cut before: rising, with gaps, shuffled within the older half
    position = torch.randint(0, 10 ** 6, kv.shape[:3], generator=g, device=cuda_device, dtype=torch.int32)
    want = [t.clone() for t in (kv, weight, position)]
    for b in range(B):
        if lengths[b] == 0:
            continue
        slot = torch.arange(lengths[b], device=cuda_device)
        pg, off = table[b].long()[slot // page], slot % page
        for h in range(H):
            moves, _ = ref.evict(weight[pg, h, off], position[pg, h, off], budget, recent)
            if moves:
                to, frm = torch.tensor(moves, device=cuda_device).T
                for x, y in zip(want, (kv, weight, position)):
                    x[pg[to], h, off[to]] = y[pg[frm], h, off[frm]]
    new = kc.cache4_evict(kv, weight, position, table, n, budget, recent)
    assert new.tolist() == [min(m, budget) for m in lengths] and n.tolist() == lengths
    assert torch.equal(kv, want[0]) and torch.equal(position, want[2])
    assert torch.equal(weight.nan_to_num(99.0), want[1].nan_to_num(99.0))
    fa.device_status()


# ------------------------------------------------------------------ together

def step(state, x, pos):
    """One decoding step of one layer, as a program makes it: positions, append, attention with weights."""
    q, k, v = x
    q, k = ro.rotary(q, k, state["rope"], pos)
    kc.cache4_append(k, v, state["kv"], state["table"], state["lengths"], weight=state["weight"], position=state["position"], positions=pos)
    return q, kc.cache4_attention(q, state["kv"], state["table"], state["lengths"], 0.125, weight=state["weight"])


@pytest.mark.gpu
def test_prompt_then_steps_with_eviction(cuda_device):
    """A prompt through attention(), its K and V into the cache, then steps, with the cache cut back on the way."""
    dtype, B, H, D, page, S = torch.float16, 2, 4, 64, 16, 50
    table = torch.randperm(B * 8, device=cuda_device).to(torch.int32).view(B, 8)
    kv, weight, position = kc.cache4_empty(B * 8, H, page, D, device=cuda_device)
    state = {"kv": kv, "weight": weight, "position": position, "table": table, "rope": ro.rotary_table(256, D, device=cuda_device)}
    q, k, v = (rows(cuda_device, (B, H, S, D), dtype, s) for s in (1, 2, 3))
    pos = torch.arange(S, device=cuda_device, dtype=torch.int32).expand(B, S).contiguous()
    qr, kr = ro.rotary(q, k, state["rope"], pos)
    o = fa.attention(qr, kr, v, True, 0.125, 128, 128)
    state["lengths"] = torch.full((B,), S, dtype=torch.int32, device=cuda_device)
    kc.cache4_append(kr, v, kv, table, state["lengths"], weight=weight, position=position, positions=pos)
    # the same prompt over the cache: attention() on what the cache stands for, in one more rounding of K and V
    ck, cv = kc.cache4_read(kv, table, state["lengths"], S, dtype)
    oc = kc.cache4_attention(qr, kv, table, state["lengths"], 0.125, weight=weight)
    assert torch.allclose(oc.float(), fa.attention(qr, ck, cv, True, 0.125, 128, 128).float(), atol=1e-2, rtol=1e-2)
    assert float((oc.float() - o.float()).norm() / o.float().norm()) < 0.3      # 4 bits: a sanity bound, no accuracy claim
    assert abs(float(weight.sum()) - B * H * S) < 1e-2                          # a softmax row adds one
    for i in range(20):
        state["lengths"] = state["lengths"] + 1
        x = [rows(cuda_device, (B, H, 1, D), dtype, 100 + 3 * i + j) for j in range(3)]
        before = weight.clone()
        now = torch.full((B, 1), S + i, dtype=torch.int32, device=cuda_device)
        qs, os = step(state, x, now)
        for b in range(B):                                                      # append has cleared the new token's weight
            last = int(state["lengths"][b]) - 1
            before[table[b, last // page], :, last % page] = 0
        check_attention(os, qs, kv, table, state["lengths"], 0.125, None, None, weight, before)
        if i % 4 == 3:
            state["lengths"] = kc.cache4_evict(kv, weight, position, table, state["lengths"], 40, 8)
            assert state["lengths"].tolist() == [40, 40]
            held = position[table[0, :3].long()].transpose(0, 1).reshape(H, -1)[:, :40]
            for h in range(H):
                assert set(range(S + i - 7, S + i + 1)) <= set(held[h].tolist()) and len(set(held[h].tolist())) == 40
    fa.device_status()


@pytest.mark.gpu
def test_a_captured_step_replays_with_other_lengths(cuda_device):
    dtype, B, H, D, page = torch.bfloat16, 3, 2, 128, 32
    kv, table, lengths = make(cuda_device, [60, 0, 31], H, D, page, dtype, room=96)
    kv[:] = torch.where(kv == 255, torch.zeros_like(kv), kv)
    state = {"kv": kv, "weight": torch.zeros(kv.shape[:3], device=cuda_device), "position": torch.zeros(kv.shape[:3], dtype=torch.int32, device=cuda_device),
             "table": table, "lengths": lengths, "rope": ro.rotary_table(128, D, device=cuda_device)}
    x = [rows(cuda_device, (B, h, 1, D), dtype, h) for h in (4, 2, 2)]
    pos = torch.zeros(B, 1, dtype=torch.int32, device=cuda_device)
    saved = {n: state[n].clone() for n in ("kv", "weight", "position")}

    def reset(ls, p):
        for n, t in saved.items():
            state[n].copy_(t)
        lengths.copy_(torch.tensor(ls))
        pos.fill_(p)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(state, x, pos)
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for _ in range(2):                                              # two graphs of the same state
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(state, x, pos)[1]
            new = kc.cache4_evict(kv, state["weight"], state["position"], table, lengths, 64, 4)
        graphs.append((graph, out, new))
    for ls, p in (([61, 1, 32], 5), ([90, 0, 96], 77)):
        reset(ls, p)
        want = step(state, x, pos)[1].clone()
        want_new = kc.cache4_evict(kv, state["weight"], state["position"], table, lengths, 64, 4)
        end = {n: state[n].clone() for n in saved}
        for graph, out, new in graphs:
            reset(ls, p)
            out.fill_(9)
            graph.replay()
            assert torch.equal(out, want) and torch.equal(new, want_new)
            for n in saved:
                assert torch.equal(state[n].view(torch.uint8), end[n].view(torch.uint8)), n
    fa.device_status()


@pytest.mark.gpu
def test_calls_on_two_streams(cuda_device):
    dtype, H, D = torch.float16, 2, 128
    sets = [make(cuda_device, [2000 + 100 * i, 40], H, D, 64, dtype, seed=i) for i in range(2)]
    q = [rows(cuda_device, (2, 8, 1, D), dtype, i) for i in range(2)]
    want = [kc.cache4_attention(q[i], *sets[i], 0.1) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kc.cache4_attention(q[i], *sets[i], 0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.gpu
def test_refusals_on_the_device(cuda_device):
    dtype = torch.float16
    kv, table, n = make(cuda_device, [20, 5], 2, 64, 16, dtype)
    q, weight = torch.zeros(2, 4, 1, 64, dtype=dtype, device=cuda_device), torch.zeros(kv.shape[:3], device=cuda_device)
    k = q[:, :2]
    position = torch.zeros(kv.shape[:3], dtype=torch.int32, device=cuda_device)
    for call in (lambda: kc.cache4_attention(q[:, :3], kv, table, n, 0.1), lambda: kc.cache4_attention(q.float(), kv, table, n, 0.1),
                 lambda: kc.cache4_attention(q[..., :32], kv, table, n, 0.1), lambda: kc.cache4_attention(q[:1], kv, table, n, 0.1),
                 lambda: kc.cache4_attention(q, kv[:, :, ::2], table, n, 0.1), lambda: kc.cache4_attention(q, kv, table.long(), n, 0.1),
                 lambda: kc.cache4_attention(q, kv, table, n.long(), 0.1), lambda: kc.cache4_attention(q, kv, table, n[:1], 0.1),
                 lambda: kc.cache4_attention(q, kv, table.cpu(), n, 0.1), lambda: kc.cache4_attention(q, kv, table.T, n, 0.1),
                 lambda: kc.cache4_attention(q, kv, table, n, 0.1, weight=weight.double()), lambda: kc.cache4_attention(q, kv, table, n, math.nan),
                 lambda: kc.cache4_attention(q, kv, table, n, 0.1, counts=n.long()), lambda: kc.cache4_append(k, k.bfloat16(), kv, table, n),
                 lambda: kc.cache4_append(q, q, kv, table, n), lambda: kc.cache4_append(k, k, kv, table, n, position=position),
                 lambda: kc.cache4_append(k, k, kv, table, n, positions=n[:, None]), lambda: kc.cache4_read(kv, table, n, 4, torch.float32),
                 lambda: kc.cache4_evict(kv, weight[:1], position, table, n, 4), lambda: kc.cache4_evict(kv, weight, weight, table, n, 4)):
        with pytest.raises(ValueError):
            call()
    assert kc.cache4_attention(q[:, :, :0], kv, table, n, 0.1).shape == (2, 4, 0, 64)
    assert kc.cache4_read(kv, table, n, 0, dtype)[0].shape == (2, 2, 0, 64)
    kc.cache4_append(k[:, :, :0], k[:, :, :0], kv, table, n)


# ------------------------------------------------------------------ the native form of the calls

@pytest.mark.gpu
def test_native_and_python_routes_agree(cuda_device, monkeypatch):
    """Ordinary calls are answered by the native code, others are not, and both give the same bits."""
    dtype, H, D, page = torch.bfloat16, 2, 64, 16
    native = ro._native
    q, k = rows(cuda_device, (2, 4, 3, D), dtype, 1), rows(cuda_device, (2, 3, H, D), dtype, 2).transpose(1, 2)
    rope = ro.rotary_table(64, D, device=cuda_device)
    pos = torch.randint(0, 64, (2, 3), device=cuda_device, dtype=torch.int32)
    counts, starts = (torch.tensor(x, dtype=torch.int32, device=cuda_device) for x in ([3, 2], [1, 0]))

    def everything():
        kv, table, n = make(cuda_device, [40, 20], H, D, page, dtype, room=60)
        weight, position = torch.zeros(kv.shape[:3], device=cuda_device), torch.zeros(kv.shape[:3], dtype=torch.int32, device=cuda_device)
        out = [*ro.rotary(q, k, rope, pos), *ro.rotary(q, k, rope, pos.long(), True), ro.rotary(q, None, rope)[0]]
        kc.cache4_append(k, k, kv, table, n, counts=counts, weight=weight, position=position, positions=pos)
        out += [*kc.cache4_read(kv, table, n, 7, dtype, starts=starts), *kc.cache4_attention(q, kv, table, n, 0.1, counts=counts, weight=weight, want_lse=True),
                kc.cache4_attention(q, kv, table, n, 0.1)]
        out += [kc.cache4_evict(kv, weight, position, table, n, 24, 5), *kc.cache4_read(kv, table, torch.clamp(n, max=24), 24, dtype), weight, position]
        return out

    seen = []
    for name in ("rotary", "cache4_append", "cache4_read", "cache4_attention", "cache4_evict"):
        fn = getattr(native, name)
        monkeypatch.setattr(native, name, lambda *a, fn=fn, name=name: seen.append((name, fn(*a))) or seen[-1][1])
    first = everything()
    assert len(seen) == 9 and all(r is not None for _, r in seen)
    monkeypatch.undo()
    monkeypatch.setattr(ro, "_native", None)
    for a, b in zip(first, everything()):
        assert torch.equal(a, b) and a.dtype == b.dtype and a.stride() == b.stride()
    # what is not ordinary
    kv, table, n = make(cuda_device, [40, 20], H, D, page, dtype, room=60)
    assert native.rotary(q.clone().requires_grad_(), k, rope, pos, False, False)[0].requires_grad
    assert native.rotary(q, k, rope.double(), pos, False, False) is None and native.rotary(q, k, rope, pos[:, :2], False, False) is None
    assert native.rotary(q[..., ::2], None, rope, None, False, False) is None and native.rotary(q, k.half(), rope, pos, False, False) is None
    assert native.cache4_attention(q, kv, table, n, 1, None, None, False) is None and native.cache4_attention(q, kv, table, n[:1], 0.1, None, None, False) is None
    assert native.cache4_attention(q[:, :3], kv, table, n, 0.1, None, None, False) is None and native.cache4_attention(q, kv[..., :64], table, n, 0.1, None, None, False) is None
    assert native.cache4_append(k, k, kv, table, n, None, None, None, pos) is None and native.cache4_append(q, q, kv, table, n, None, None, None, None) is None
    assert native.cache4_read(kv, table, n, 0, True, None) is None and native.cache4_read(kv, table.long(), n, 4, True, None) is None
    assert native.cache4_evict(kv, None, None, table, n, 4, 2) is None


@pytest.mark.gpu
def test_a_backward_pass_through_the_attention_raises(cuda_device):
    kv, table, lengths = make(cuda_device, [40], 1, 64, 16, torch.float16)
    q = rows(cuda_device, (1, 2, 1, 64), torch.float16, 7)
    want = kc.cache4_attention(q, kv, table, lengths, 0.125, want_lse=True)
    got = kc.cache4_attention(q.requires_grad_(), kv, table, lengths, 0.125, want_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(kc.cache4_attention(q, kv, table, lengths, 0.125), want[0])
    with pytest.raises(NotImplementedError):
        got[0].sum().backward()
    with torch.no_grad():
        assert not kc.cache4_attention(q, kv, table, lengths, 0.125).requires_grad


@pytest.mark.gpu
def test_scratch_is_sized_for_every_call(cuda_device):
    """The same number of slots as one sequence of two pages and as two of one page, which are different numbers of tiles; a
    table that is not contiguous, so both calls take the Python route."""
    for lengths in ([30], [16, 9]):
        kv, table, n = make(cuda_device, lengths, 1, 128, 16, torch.float16)
        wide = torch.zeros(table.shape[0], table.shape[1] + 1, dtype=torch.int32, device=cuda_device)
        wide[:, :-1] = table
        q = rows(cuda_device, (len(lengths), 1, 1, 128), torch.float16, 8)
        weight, before = (torch.zeros(kv.shape[:3], device=cuda_device) for _ in range(2))
        counts = torch.ones(2 * len(lengths), dtype=torch.int32, device=cuda_device)[::2]
        got, lse = kc.cache4_attention(q, kv, wide[:, :-1], n, 128 ** -0.5, counts=counts, weight=weight, want_lse=True)
        check_attention(got, q, kv, table, lengths, 128 ** -0.5, lse=lse, weight=weight, weight_before=before)


@pytest.mark.gpu
def test_what_follows_a_batch_without_tokens_sees_its_zeros(cuda_device):
    """No kernel of the call has work but the one that writes zeros, and the next operator waits for that one, too."""
    kv, table, lengths = make(cuda_device, [0] * 64, 2, 128, 16, torch.float16)
    q = rows(cuda_device, (64, 16, 1, 128), torch.float16, 5)
    weight = torch.zeros(kv.shape[:3], device=cuda_device)
    cos_sin, last = ro.rotary_table(4, 128, device=cuda_device), torch.tensor([3], dtype=torch.int32, device=cuda_device)
    for _ in range(20):
        stale = torch.full_like(q, math.nan)
        del stale                                                  # the next allocation of this size
        o, lse = kc.cache4_attention(q, kv, table, lengths, 0.1, weight=weight, want_lse=True)
        turned, _ = ro.rotary(o, None, cos_sin, last)
        assert bool((turned == 0).all()) and bool((o == 0).all()) and bool((lse == -math.inf).all()) and bool((weight == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,D,Hq,H,S,page,scale,std", [([46, 107, 76, 1, 275, 0, 0], 256, 80, 5, 9, 64, 1.0, 1.0),
                                                             ([5, 5, 0, 1, 2, 3, 4], 256, 4, 2, 1, 64, 0.0625, 3.0),
                                                             ([39, 1, 0, 40, 25], 128, 9, 3, 4, 128, 1.0, 3.0),
                                                             ([191, 0, 147, 1, 23], 64, 12, 3, 5, 32, -0.125, 1.0)])
def test_attention_of_few_tokens_and_many_rows(cuda_device, dtype, lengths, D, Hq, H, S, page, scale, std):
    """Rows that one token has nearly to itself, whose dims are then sums that cancel, and more rows than two blocks."""
    kv, table, n = make(cuda_device, lengths, H, D, page, dtype, seed=17, std=std)
    q = rows(cuda_device, (len(lengths), Hq, S, D), dtype, 18)
    weight = torch.rand(kv.shape[:3], device=cuda_device)
    before = weight.clone()
    got, lse = kc.cache4_attention(q, kv, table, n, scale, weight=weight, want_lse=True)
    check_attention(got, q, kv, table, lengths, scale, lse=lse, weight=weight, weight_before=before)


# ------------------------------------------------------------------ rows that see what others do not

def attention_bound(q, kv, table, lengths, scale, counts=None):
    """The result in 64 bits and the bound of check_attention, for results that are NaN in places."""
    o, _, _, (parts, middles, both, sizes, terms) = ref.attention(q, kv, table, lengths, scale, counts)
    off = 2.0 ** -19 * (1 + terms)
    return o, (HALF_STEP[q.dtype] * (o.abs() + middles) + 2.0 ** -11 * parts + 2 * off[..., None] * sizes + 2.0 ** -16 * (parts + both)
               + TINY[q.dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [32, 256])
@pytest.mark.parametrize("D,Hq", [(64, 1), (64, 8), (128, 4), (128, 16), (256, 2)])
def test_a_row_of_v_with_an_infinity_beside_one_of_wide_scales(cuda_device, dtype, bad, D, Hq):
    """The last of two query tokens sees slot 8, whose V holds an infinity in its first `bad` dims; both rest on slot 0, whose
    V is a hundred times as wide as the others'.  The first has finite results, the second NaN in the groups of these dims only."""
    n = 9
    kv, weight, position = kc.cache4_empty(2, 1, 16, D, device=cuda_device)
    table, lengths = torch.tensor([[1]], dtype=torch.int32, device=cuda_device), torch.tensor([n], dtype=torch.int32, device=cuda_device)
    k, v, q = (rows(cuda_device, s, dtype, i) for i, s in enumerate(((1, 1, n, D), (1, 1, n, D), (1, Hq, 2, D))))
    k[:, :, 0, 0], q[..., 0] = 8, 8
    v[:, :, 0] *= 100
    v[:, :, 8, : bad : 32] = math.inf
    kc.cache4_append(k, v, kv, table, lengths)
    got = kc.cache4_attention(q, kv, table, lengths, 0.5)
    check_attention(got[:, :, :1], q[:, :, :1], kv, table, [n - 1], 0.5)
    o, bound = attention_bound(q, kv, table, lengths, 0.5)
    nan = torch.zeros_like(o, dtype=torch.bool)
    nan[:, :, 1, :bad] = True
    assert torch.equal(o.isnan(), nan) and torch.equal(got.isnan(), nan)
    assert bool(((got.double() - o).abs() <= bound)[~nan].all())
    fa.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,Hq,H,S", [(64, 4, 4, 1), (64, 24, 2, 1), (128, 8, 2, 1), (128, 16, 2, 2), (256, 4, 2, 3)])
def test_values_with_a_common_offset(cuda_device, dtype, D, Hq, H, S):
    """V rows that are nearly the same come back as what they have in common: the weights of the groups' middles and the sum that
    they are divided by are the same to 2^-16, so that the result's own rounding, half a step at its size, is what is left."""
    lengths = [3, 4, 5, 9, 40, 700]
    B, n = len(lengths), max(lengths)
    kv, table, ls = make(cuda_device, lengths, H, D, 16, dtype, seed=3)
    k = rows(cuda_device, (B, H, n, D), dtype, 1)
    offset = (1 + torch.rand((B, H, 1, D // 32, 1), generator=torch.Generator(device=cuda_device).manual_seed(2), device=cuda_device)).expand(-1, -1, n, -1, 32).flatten(3)
    v = (offset + 2.0 ** -6 * rows(cuda_device, (B, H, n, D), torch.float32, 3)).to(dtype)
    kc.cache4_append(k, v, kv, table, ls, counts=ls)
    q = rows(cuda_device, (B, Hq, S, D), dtype, 4)
    got = kc.cache4_attention(q, kv, table, ls, 0.1)
    o, _, _, (parts, middles, both, sizes, terms) = ref.attention(q, kv, table, ls, 0.1)
    rest = 2.0 ** -11 * parts + 2.0 ** -16 * (parts + middles + both) + 2.0 ** -18 * (1 + terms)[..., None] * sizes
    half = 2.0 ** torch.floor(torch.log2(o.abs() + rest)) * HALF_STEP[dtype]
    err = (got.double() - o).abs()
    assert bool((err <= half + rest).all()), (float((err - half - rest).max()), int((err > half + rest).sum()), err.numel())


@pytest.mark.gpu
def test_a_tangent_through_the_attention_raises(cuda_device):
    """As one through attention() does: nothing would be said of its derivative otherwise."""
    kv, table, lengths = make(cuda_device, [40], 1, 64, 16, torch.float16)
    q = rows(cuda_device, (1, 2, 1, 64), torch.float16, 7)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError):
            kc.cache4_attention(dual, kv, table, lengths, 0.125)
        with pytest.raises(NotImplementedError), torch.no_grad():
            kc.cache4_attention(dual, kv, table, lengths, 0.125)
        with pytest.raises(NotImplementedError):
            kc.cache4_attention(forward_ad.make_dual(q.clone().requires_grad_(), torch.ones_like(q)), kv, table, lengths, 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("length,counts", [(49, None), (50, [3, 3]), (51, None), (52, None), (2 ** 31 - 1, None), (48 + 2, [1, 1]), (-1, None)])
def test_append_beyond_the_pages_keeps_what_they_hold(cuda_device, length, counts):
    """Rows whose slots would be behind the last page are left out, and the rows in front of them keep what they are."""
    dtype, H, D, page, S, room = torch.bfloat16, 2, 64, 16, 3, 48
    kv, table, lengths = make(cuda_device, [room, 20], H, D, page, dtype)
    weight, position = torch.rand(kv.shape[:3], device=cuda_device), torch.zeros(kv.shape[:3], dtype=torch.int32, device=cuda_device)
    lengths[0] = length
    k, v = rows(cuda_device, (2, H, S, D), dtype, 1), rows(cuda_device, (2, H, S, D), dtype, 2)
    positions = torch.full((2, S), 9, dtype=torch.int32, device=cuda_device)
    want = [t.clone() for t in (kv, weight, position)]
    for b, n in enumerate((length, 20)):
        c = S if counts is None else counts[b]
        for j in range(c):
            slot = n - c + j
            if 0 <= slot < room:
                at = (int(table[b, slot // page]), slice(None), slot % page)
                want[0][at] = ref.records(k[b, :, j], v[b, :, j])
                want[1][at], want[2][at] = 0.0, 9
    fa.device_status()
    c = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=cuda_device)
    kc.cache4_append(k, v, kv, table, lengths, counts=c, weight=weight, position=position, positions=positions)
    with pytest.raises(RuntimeError, match="device status 0x20003"):
        fa.device_status()
    for got, exp in zip((kv, weight, position), want):
        assert torch.equal(got, exp)


@pytest.mark.gpu
@pytest.mark.parametrize("route", ["native", "python"])
@pytest.mark.parametrize("budget", [2 ** 31 - 1, 1024, 1 << 12, (1 << 12) - 1])
def test_scratch_of_an_eviction_goes_by_what_can_move(cuda_device, monkeypatch, route, budget):
    """A budget at or above what the table has room for moves nothing, one a slot below it one record per head at most."""
    if route == "python":
        monkeypatch.setattr(ro, "_native", None)
    B, H, D, page, n = 2, 4, 64, 64, 1 << 12
    kv, weight, position = kc.cache4_empty(B * n // page, H, page, D, device=cuda_device)
    table = torch.arange(B * n // page, dtype=torch.int32, device=cuda_device).view(B, -1)
    lengths = torch.tensor([n, 100], dtype=torch.int32, device=cuda_device)
    kv.random_(0, 256)
    weight.random_(1, 1000)
    position.copy_(torch.arange(B * n, dtype=torch.int32, device=cuda_device).view(-1, 1, page).expand_as(position))
    want = kv.clone()
    slot = torch.arange(n, device=cuda_device)
    for h in range(H):
        moves, _ = ref.evict(weight[:n // page, h].flatten(), slot, budget, 5)
        for to, source in moves:
            want[to // page, h, to % page] = kv[source // page, h, source % page]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    new = kc.cache4_evict(kv, weight, position, table, lengths, budget, 5)
    most = min(budget, max(n - budget, 0))
    assert torch.cuda.max_memory_allocated() - before <= B * H * 8 * (most + 2) + 2048
    assert new.tolist() == [min(n, budget), 100] and torch.equal(kv, want)
    fa.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D,Hq,H", [(64, 4, 4), (128, 8, 2)])
def test_weights_of_tokens_that_a_nan_row_does_not_see(cuda_device, wide, D, Hq, H):
    """The first of two query tokens is NaN: the tokens that it sees get NaN, the last one the second token's weight alone.  With
    scores that are kept and, for a table far wider than the cache, ones that are computed again."""
    n, page = 37, 16
    kv, table, lengths = make(cuda_device, [n], H, D, page, torch.float16)
    if wide:
        table = torch.cat((table, torch.full((1, 4096), -1, dtype=torch.int32, device=cuda_device)), 1)
    q = rows(cuda_device, (1, Hq, 2, D), torch.float16, 1)
    weight, want = (torch.zeros(kv.shape[:3], device=cuda_device) for _ in range(2))
    kc.cache4_attention(q, kv, table, lengths, 0.1, weight=want)
    last = (int(table[0, (n - 1) // page]), slice(None), (n - 1) % page)
    want, weight = want[last].clone(), torch.zeros_like(weight)
    q[:, :, 0, 3] = math.nan
    kc.cache4_attention(q, kv, table, lengths, 0.1, weight=weight)
    slot = torch.arange(n - 1, device=cuda_device)
    assert bool(weight[table[0].long()[slot // page], :, slot % page].isnan().all())
    assert torch.equal(weight[last], want) and bool((want > 0).all())


def test_the_workspace_query_refuses_what_the_call_refuses():
    too_large = _capi.RSFA_ERR_TOO_LARGE
    assert lib.rsfa_cache4_attention_workspace(c_cache(), 64, 1 << 30) == too_large
    assert lib.rsfa_cache4_attention_workspace(c_cache(batch=1 << 20, max_pages=1 << 26, table_stride=0), 2, 4) == too_large
    p = ctypes.c_void_p(4096)
    assert lib.rsfa_cache4_evict_workspace(1 << 16, 1 << 15, 8) == too_large
    assert lib.rsfa_cache4_evict_workspace(1 << 16, (1 << 15) - 1, (1 << 31) - 1) == too_large
    c = c_cache(batch=1 << 16, heads=(1 << 15) - 1, max_pages=1 << 26, table_stride=0, kv_stride=(1 << 40, 1280), weight_stride=(1 << 20, 16), position_stride=(1 << 20, 16))
    assert lib.rsfa_cache4_evict(c, 1 << 29, 2, ctypes.c_void_p(8192), p, 1 << 62, None) == too_large


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size", [(torch.float16, 2.0 ** 12), (torch.bfloat16, 2.0 ** 40), (torch.bfloat16, 2.0 ** 100), (torch.bfloat16, 2.0 ** -60)])
@pytest.mark.parametrize("at", [0, 0.6, 1])
@pytest.mark.parametrize("D,Hq,n", [(64, 2, 9), (64, 8, 300), (128, 3, 9), (128, 8, 300), (128, 16, 20000), (256, 2, 9), (256, 2, 150)])
def test_a_row_of_v_of_another_size(cuda_device, dtype, size, at, D, Hq, n):
    """One slot's V is `size` times as large as the others.  The second of two query tokens gives it no weight in its even heads (a
    score far below the others) and rests on it in the odd ones; the first weighs it like any other, or does not see it where it
    is the last.  Each result is as good as if there were no other rows."""
    pages, slot = n // 16 + 1, int(at * (n - 1))
    kv, weight, position = kc.cache4_empty(pages, 1, 16, D, device=cuda_device)
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    lengths = torch.tensor([n], dtype=torch.int32, device=cuda_device)
    k, v, q = (rows(cuda_device, s, dtype, i) for i, s in enumerate(((1, 1, n, D), (1, 1, n, D), (1, Hq, 2, D))))
    k[:, :, slot, 0] = 100
    q[..., 0] = 0
    q[:, ::2, 1, 0], q[:, 1::2, 1, 0] = -20, 20
    v[:, :, slot] *= size
    kc.cache4_append(k, v, kv, table, lengths)
    got, lse = kc.cache4_attention(q, kv, table, lengths, 1.0, want_lse=True)
    o, bound = attention_bound(q, kv, table, lengths, 1.0)
    widest = ref.records(k.reshape(n, D), v.reshape(n, D))[:, -(D // 8):].contiguous().view(dtype)[:, ::2].max()
    if size < 1:
        # A product p * s that is no more than half of fp16's smallest step, 2^-25, is lost, times |u - 8| <= 8, where the weights
        # add up to 2^10 at least, in units of the widest scale at most: a row of small values is as good as these allow.
        bound = bound + n * 2.0 ** -32 * float(widest)
    assert bool(((got.double() - o).abs() <= bound).all())
    # A code is an fp16 number below 2^-14, a query's largest element one of 2^10 to 2^11, and an MMA cuts 16 products and their
    # sum so far off at 2^-24 of what these exponents allow, 2^-3: a score is off by 17 * 2^-27 for codes that count 2^-24 and
    # queries that count 2^-10 of their largest, once for the codes at the bottom and 1/16 of it for the others, per group.
    _, want, _, (_, _, _, _, terms) = ref.attention(q, kv, table, lengths, 1.0)
    scales = ref.records(k.reshape(n, D), v.reshape(n, D))[:, D:D + D // 8].contiguous().view(dtype)[:, ::2].double()
    cut = 18.1 * 2.0 ** -13 * q.double().abs().amax(-1) * scales.sum(-1).max()
    assert bool(((lse.double() - want).abs() <= 2.0 ** -19 * (1 + terms) + cut + 2.0 ** -22 * want.abs() + 2.0 ** -20).all())


# ------------------------------------------------------------------ shares of many tiles

@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype,D,Hq,S,lengths", [
    (torch.float16, 64, 16, 1, [41000, 31000, 0, 77]), (torch.bfloat16, 128, 32, 2, [31000, 77, 41000]), (torch.bfloat16, 64, 160, 1, [30000, 18000]),
    (torch.float16, 128, 96, 2, [5, 30000, 0, 18000]), (torch.float16, 256, 32, 1, [30000, 18000, 2]),
])
def test_shares_longer_than_a_window_of_pages(cuda_device, wide, dtype, D, Hq, S, lengths):
    """Sixteen heads in pages of 16 slots: a warp's share (of 148 multiprocessors with twelve of them each, eight at D = 256 or with
    more than eight rows) is 40 pages and more, so that the window of 32 page numbers moves on, every slot of the ring is used again and
    again, and the weights take several rounds.  Three of the heads are compared."""
    H, page, heads = 16, 16, [0, 5, 15]
    assert H * sum(lengths) / 16 / (148 * (8 if D == 256 or Hq // H * S > 8 else 12)) > 40
    kv, table, n = make(cuda_device, lengths, H, D, page, dtype, seed=5)
    if wide:
        table = torch.cat((table, torch.full((len(lengths), 4 * table.shape[1]), -1, dtype=torch.int32, device=cuda_device)), 1)
    q = rows(cuda_device, (len(lengths), Hq, S, D), dtype, 6, 2.0)
    before = torch.rand(kv.shape[:3], device=cuda_device)
    weight = before.clone()
    o, lse = kc.cache4_attention(q, kv, table, n, 0.1, weight=weight, want_lse=True)
    assert torch.equal(kc.cache4_attention(q, kv, table, n, 0.1), o)
    some = [x.unflatten(1, (H, Hq // H))[:, heads].flatten(1, 2) for x in (o, q, lse)]
    check_attention(some[0], some[1], kv[:, heads], table, n, 0.1, None, some[2], weight[:, heads], before[:, heads])
    fa.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype,D,Hq,H,S", [(torch.float16, 64, 4, 2, 1), (torch.bfloat16, 128, 8, 2, 1), (torch.float16, 128, 24, 2, 1), (torch.bfloat16, 256, 2, 2, 2)])
def test_shares_of_several_heads_and_sequences(cuda_device, wide, dtype, D, Hq, H, S):
    """2000 ragged sequences: a warp's share goes from the last head of one to the heads of the next ones, past some without
    tokens, and the second head of a short one has the pages of the first.  Every fortieth sequence is compared."""
    B, page, n = 2000, 16, 260
    g = torch.Generator(device=cuda_device).manual_seed(1)
    lengths = torch.tensor([0, 1, 2, 5, 16, 33, 100, 260], dtype=torch.int32, device=cuda_device)[torch.randint(0, 8, (B,), generator=g, device=cuda_device)]
    each = -(-n // page)
    kv = torch.full((B * each + 3, H, page, 5 * D // 4), 255, dtype=torch.uint8, device=cuda_device)
    table = torch.randperm(B * each + 3, generator=g, device=cuda_device)[: B * each].to(torch.int32).view(B, each)
    k, v = (rows(cuda_device, (B, H, n, D), dtype, s) for s in (2, 3))
    kc.cache4_append(k, v, kv, table, lengths, counts=lengths)
    if wide:
        table = torch.cat((table, torch.full((B, 4 * each), -1, dtype=torch.int32, device=cuda_device)), 1)
    q = rows(cuda_device, (B, Hq, S, D), dtype, 6, 2.0)
    before = torch.rand(kv.shape[:3], device=cuda_device)
    weight = before.clone()
    o, lse = kc.cache4_attention(q, kv, table, lengths, 0.1, weight=weight, want_lse=True)
    assert torch.equal(kc.cache4_attention(q, kv, table, lengths, 0.1), o)
    some = torch.arange(0, B, 40, device=cuda_device)
    theirs = table[some, :each].long().flatten()
    only = before.clone()
    only[theirs] = weight[theirs]
    check_attention(o[some], q[some], kv, table[some], lengths[some], 0.1, None, lse[some], only, before)
    empty = lengths == 0
    assert bool((o[empty] == 0).all()) and bool((lse[empty] == -math.inf).all()) and bool(torch.isfinite(o).all())
    # every row of a softmax adds one to a head's tokens
    seen = torch.minimum(lengths, torch.full_like(lengths, S)).sum()
    assert abs(float((weight.double() - before.double()).sum()) - float(seen) * Hq) <= 2.0 ** -19 * 64 * float(seen) * Hq
    fa.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("length,budget,recent", [(33000, 500, 100), (50001, 4000, 0), (65536, 1, 1)])
def test_evict_of_more_pages_than_are_kept_at_hand(cuda_device, length, budget, recent):
    """Sequences of more than 2048 pages, which select looks up again in the table, and of more keys than shared memory holds."""
    H, D, page = 2, 64, 16
    pages = -(-length // page)
    g = torch.Generator(device=cuda_device).manual_seed(9)
    table = torch.randperm(2 * pages, generator=g, device=cuda_device)[:pages].to(torch.int32)[None]
    kv = torch.randint(0, 256, (2 * pages, H, page, 5 * D // 4), generator=g, device=cuda_device, dtype=torch.uint8)
    weight = torch.rand(kv.shape[:3], generator=g, device=cuda_device)
    position = torch.randint(0, 10 ** 6, kv.shape[:3], generator=g, device=cuda_device, dtype=torch.int32)
    want = [t.clone() for t in (kv, weight, position)]
    slot = torch.arange(length, device=cuda_device)
    pg, off = table[0].long()[slot // page], slot % page
    for h in range(H):
        moves, _ = ref.evict(weight[pg, h, off], position[pg, h, off], budget, recent)
        if moves:
            to, frm = torch.tensor(moves, device=cuda_device).T
            for x, y in zip(want, (kv, weight, position)):
                x[pg[to], h, off[to]] = y[pg[frm], h, off[frm]]
    new = kc.cache4_evict(kv, weight, position, table, torch.tensor([length], dtype=torch.int32, device=cuda_device), budget, recent)
    assert new.tolist() == [budget]
    for got, exp in zip((kv, weight, position), want):
        assert torch.equal(got, exp)
    fa.device_status()
