"""Rows into a paged cache of 8-bit codes (or fp16) and back: quantised write, read, and the
norm + rotary + write pass, against plain 64-bit forms."""
import numpy as np
import pytest

from _cache8 import E32, H16, NAME, TOP, code_dtype, half_step, norm_rope, norm_rope_bound, values
from _helpers import dev, host, say
from kvcache_amd import KVC_E4M3, KVC_F16, KVC_F32, KVC_I8, ops
from kvcache_amd.device import DeviceBuffer, Stream

pytestmark = pytest.mark.gpu


def _slots(rng, rows, block, nb, skip=0.0):
    s = rng.permutation(nb * block)[:rows].astype(np.int32)
    s[rng.random(rows) < skip] = -1
    return s


def _at(pool, slots, block):
    """Rows [rows, Hkv, ...] of a pool [nb, Hkv, block, ...] at slots >= 0."""
    return pool[slots // block, :, slots % block]


def _write(k, v, slots, nb, Hkv, D, block, dtype, kv_dtype, stream=None):
    kp = np.full((nb, Hkv, block, D), 77, code_dtype(kv_dtype))
    sc = np.full((nb, Hkv, block, 2), 5.0, np.float32)
    dk, dv, ds = dev(kp), dev(kp + 1), dev(sc)
    ops.write_kv_q8(dev(k), dev(v), dk, dv, ds, dev(slots), len(k), Hkv, D, block, dtype=dtype, kv_dtype=kv_dtype,
                    stream=stream)
    return (host(dk, kp.dtype, kp.shape), host(dv, kp.dtype, kp.shape), host(ds, np.float32, sc.shape)), (dk, dv, ds)


@pytest.mark.parametrize("kv_dtype", [KVC_I8, KVC_E4M3], ids=NAME.get)
@pytest.mark.parametrize("rows,Hkv,D,block,dtype", [
    (1, 1, 32, 16, KVC_F16), (7, 2, 64, 16, KVC_F16), (33, 3, 128, 5, KVC_F32), (129, 8, 128, 16, KVC_F16),
    (65, 2, 256, 32, KVC_F16), (200, 5, 64, 1, KVC_F32), (1000, 1, 32, 24, KVC_F32)])
def test_quantised_write_and_read(rows, Hkv, D, block, dtype, kv_dtype):
    say(f"write_kv_q8 rows={rows} Hkv={Hkv} D={D} block={block} dtype={dtype} {NAME[kv_dtype]}")
    rng = np.random.default_rng(rows + D)
    t = np.float16 if dtype == KVC_F16 else np.float32
    k, v = ((rng.standard_normal((rows, Hkv, D)) * np.exp(rng.standard_normal((rows, Hkv, 1)))).astype(t) for _ in "kv")
    k[0] = 0                     # a zero row: scale 0, codes 0
    v[-1, 0, 1:] = 0             # one value alone is the largest code
    nb = -(-rows // block) + 3
    slots = _slots(rng, rows, block, nb, 0.2)
    (kp, vp, sc), bufs = _write(k, v, slots, nb, Hkv, D, block, dtype, kv_dtype)
    on = slots >= 0
    off = np.ones(nb * block, bool)
    off[slots[on]] = False
    for pool, base in ((kp, 77), (vp, 78)):  # slots that no row names are left as they were
        assert (pool.transpose(0, 2, 1, 3).reshape(nb * block, -1)[off] == base).all()
    assert (sc.transpose(0, 2, 1, 3).reshape(nb * block, -1)[off] == 5).all()
    for i, (x, pool) in enumerate(((k, kp), (v, vp))):
        x = x[on].astype(np.float64)
        s = _at(sc, slots[on], block)[..., i].astype(np.float64)
        c = values(_at(pool, slots[on], block), kv_dtype)
        want = np.abs(x).max(-1) / TOP[kv_dtype]
        assert np.abs(s - want).max(initial=0) <= (want * 2.0 ** -23).max(initial=0)
        assert not (c[s == 0]).any()
        # the code is the nearest but where x / s lies within its fp32 error (3 roundings) of a tie
        y = x / np.where(want > 0, want, 1)[..., None]
        err = np.abs(c - y)
        assert (err <= half_step(y, 1.0, kv_dtype) + np.abs(y) * 4 * E32).all()
    # read back: one fp32 product, then one rounding to the rows' type
    for out_t, out_d in ((np.float16, KVC_F16), (np.float32, KVC_F32)):
        ko, vo = dev(np.full(k.shape, 9, out_t)), dev(np.full(k.shape, 9, out_t))
        ops.read_kv(ko, vo, *bufs, dev(slots), rows, Hkv, D, block, dtype=out_d, kv_dtype=kv_dtype)
        for i, (buf, pool) in enumerate(((ko, kp), (vo, vp))):
            got = host(buf, out_t, k.shape)
            assert (got[~on] == 9).all()
            c = values(_at(pool, slots[on], block), kv_dtype).astype(np.float32)
            assert (got[on] == (c * _at(sc, slots[on], block)[..., i][..., None]).astype(out_t)).all()


@pytest.mark.parametrize("kv_dtype", [KVC_I8, KVC_E4M3], ids=NAME.get)
def test_rows_that_are_not_finite_or_tiny(kv_dtype):
    say(f"write_kv_q8 with Inf, NaN and tiny rows, {NAME[kv_dtype]}")
    Hkv, D, block = 2, 64, 16
    k = np.random.default_rng(0).standard_normal((6, Hkv, D)).astype(np.float32)
    k[0, 0, 3], k[1, 1, 63], k[2, 0, 0] = np.inf, np.nan, -np.inf
    k[3] *= 1e-35                # below 2^-100: zeros
    k[4] *= 1e-29                # above it: held
    k[5, 0] = np.float32(3e38)
    slots = np.arange(6, dtype=np.int32)
    (kp, vp, sc), bufs = _write(k, k, slots, 1, Hkv, D, block, KVC_F32, kv_dtype)
    bad = np.zeros((6, Hkv), bool)
    bad[0, 0] = bad[1, 1] = bad[2, 0] = True
    for i, pool in enumerate((kp, vp)):
        c, s = values(_at(pool, slots, block), kv_dtype), _at(sc, slots, block)[..., i]
        assert (np.isnan(s) == bad).all() and not c[bad].any() and np.isfinite(c).all()
        assert not s[3].any() and not c[3].any()
        x = k[~bad].astype(np.float64)
        keep = np.abs(x).max(-1) > 1e-30
        assert (np.abs(c[~bad][keep] * s[~bad][keep][:, None] - x[keep]) <=
                half_step(x[keep], s[~bad][keep][:, None].astype(np.float64), kv_dtype) * 1.001).all()
    ko = dev(np.zeros(k.shape, np.float32))
    ops.read_kv(ko, dev(np.zeros(k.shape, np.float32)), *bufs, dev(slots), 6, Hkv, D, block, dtype=KVC_F32,
                kv_dtype=kv_dtype)
    assert (np.isnan(host(ko, np.float32, k.shape)).all(-1) == bad).all()


def test_read_of_an_fp16_cache():
    say("read_kv fp16")
    rng = np.random.default_rng(2)
    kp, vp = (rng.standard_normal((5, 3, 16, 128)).astype(np.float16) for _ in "kv")
    kp[1, 2, 3, 4] = np.inf
    slots = _slots(rng, 40, 16, 5, 0.1)
    for t, d in ((np.float16, KVC_F16), (np.float32, KVC_F32)):
        ko, vo = dev(np.full((40, 3, 128), 2, t)), dev(np.full((40, 3, 128), 2, t))
        ops.read_kv(ko, vo, dev(kp), dev(vp), None, dev(slots), 40, 3, 128, 16, dtype=d, kv_dtype=KVC_F16)
        for buf, pool in ((ko, kp), (vo, vp)):
            got = host(buf, t, (40, 3, 128))
            assert (got[slots >= 0] == _at(pool, slots[slots >= 0], 16).astype(t)).all()
            assert (got[slots < 0] == 2).all()


def _norm_rope_write(x, pos, slots, Hq, Hkv, D, block, nb, kv_dtype, qn, kn, theta, eps, stride, stream=None):
    M = len(x)
    wide = np.full((M, stride), 9.0, np.float16)
    wide[:, : (Hq + 2 * Hkv) * D] = x.reshape(M, -1)
    kp = np.zeros((nb, Hkv, block, D), code_dtype(kv_dtype))
    sc = np.zeros((nb, Hkv, block, 2), np.float32)
    q, dk, dv, ds = dev(np.zeros((M + 1, Hq, D), np.float16)), dev(kp), dev(kp), dev(sc)
    args = (q, dk, dv, None if kv_dtype == KVC_F16 else ds, dev(wide), dev(pos), dev(slots), M, Hq, Hkv, D, block, theta)
    keep = [dev(w) if w is not None else None for w in (qn, kn)]
    ops.qk_norm_rope_write(*args, row_stride=stride, q_norm=keep[0], k_norm=keep[1], eps=eps, kv_dtype=kv_dtype,
                           stream=stream)
    if stream is not None:
        from kvcache_amd.device import synchronize
        synchronize()
    return (host(q, np.float16, (M + 1, Hq, D)), host(dk, kp.dtype, kp.shape), host(dv, kp.dtype, kp.shape),
            host(ds, np.float32, sc.shape))


@pytest.mark.parametrize("kv_dtype", [KVC_F16, KVC_I8, KVC_E4M3], ids=NAME.get)
@pytest.mark.parametrize("M,Hq,Hkv,D,block,norm,extra", [
    (1, 14, 2, 64, 16, True, 0), (5, 8, 8, 64, 16, True, 8), (33, 32, 8, 128, 16, True, 0), (70, 3, 1, 32, 7, False, 64),
    (17, 6, 2, 256, 32, True, 0), (300, 4, 4, 128, 16, False, 0), (9, 64, 1, 64, 16, True, 24)])
def test_norm_rope_write(M, Hq, Hkv, D, block, norm, extra, kv_dtype):
    say(f"qk_norm_rope_write M={M} Hq={Hq} Hkv={Hkv} D={D} block={block} norm={norm} {NAME[kv_dtype]}")
    rng = np.random.default_rng(M + Hq)
    heads = Hq + 2 * Hkv
    x = (rng.standard_normal((M, heads, D)) * 0.7).astype(np.float16)
    x[0, 0] = 0  # a zero row stays zero through the norm
    pos = rng.integers(0, [2, 4096, 1 << 20, (1 << 31) - 1][M % 4], M).astype(np.int32)
    pos[0] = 0
    nb = -(-M // block) + 2
    slots = _slots(rng, M, block, nb, 0.15)
    qn, kn = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float16) if norm else None for _ in "qk")
    theta, eps = 1e4 if M % 2 else 1e6, 1e-6
    q, kp, vp, sc = _norm_rope_write(x, pos, slots, Hq, Hkv, D, block, nb, kv_dtype, qn, kn, theta, eps,
                                     heads * D + extra)
    want, size = norm_rope(x[:, :Hq], qn, eps, pos, theta)
    assert not q[M].any()  # rows behind the last one are left as they were
    assert (np.abs(q[:M] - want) <= np.abs(want) * H16 + norm_rope_bound(size, D) + 2.0 ** -25).all()
    on = slots >= 0
    kwant, ksize = norm_rope(x[:, Hq:Hq + Hkv], kn, eps, pos, theta)
    kerr = norm_rope_bound(ksize, D)
    vwant = x[:, Hq + Hkv:].astype(np.float64)
    off = np.ones(nb * block, bool)
    off[slots[on]] = False
    for i, (pool, w, e) in enumerate(((kp, kwant, kerr), (vp, vwant, 0 * vwant))):
        assert not pool.transpose(0, 2, 1, 3).reshape(nb * block, -1)[off].any()
        w, e = w[on], e[on]
        c = values(_at(pool, slots[on], block), kv_dtype)
        if kv_dtype == KVC_F16:
            assert (np.abs(c - w) <= np.abs(w) * H16 + e + 2.0 ** -25).all()
            continue
        s = _at(sc, slots[on], block)[..., i].astype(np.float64)
        top = np.abs(w).max(-1)
        assert (np.abs(s - top / TOP[kv_dtype]) <= top / TOP[kv_dtype] * 2.0 ** -23 + e.max(-1) / TOP[kv_dtype]).all()
        # half a step of the code, the value's own fp32 error and that of the quotient
        assert (np.abs(c * s[..., None] - w) <= half_step(w, s[..., None], kv_dtype) * (1 + 2.0 ** -12) + 2 * e +
                np.abs(w) * 4 * E32).all()


def test_norm_rope_write_on_its_own_stream_repeats_its_bits():
    say("qk_norm_rope_write twice, the second time on a stream of its own")
    rng = np.random.default_rng(3)
    M, Hq, Hkv, D = 40, 8, 2, 128
    x = rng.standard_normal((M, Hq + 2 * Hkv, D)).astype(np.float16)
    pos, slots = np.arange(M, dtype=np.int32), rng.permutation(48)[:M].astype(np.int32)
    st = Stream()
    a, b = (_norm_rope_write(x, pos, slots, Hq, Hkv, D, 16, 3, KVC_I8, None, None, 1e4, 1e-6, (Hq + 2 * Hkv) * D, s)
            for s in (None, st.handle))
    assert all((u == w).all() for u, w in zip(a, b))


@pytest.mark.parametrize("kv_dtype", [KVC_I8, KVC_E4M3], ids=NAME.get)
def test_pool_offsets_past_32_bits(kv_dtype):
    """A pool of more than 2^32 bytes: the last block's rows are written and read at their place."""
    say(f"write_kv_q8 past 4 GiB, {NAME[kv_dtype]}")
    Hkv, D, block = 8, 128, 16
    nb = (1 << 32) // (Hkv * D * block) + 5
    kp, vp, sc = (DeviceBuffer(nb * Hkv * block * n) for n in (D, D, 8))
    for b in (kp, vp, sc):
        b.zero()
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((20, Hkv, D)).astype(np.float16) for _ in "kv")
    slots = (nb * block - 1 - np.arange(20)).astype(np.int32)
    slots[7] = 3
    ops.write_kv_q8(dev(k), dev(v), kp, vp, sc, dev(slots), 20, Hkv, D, block, kv_dtype=kv_dtype)
    ko, vo = dev(np.zeros(k.shape, np.float32)), dev(np.zeros(k.shape, np.float32))
    ops.read_kv(ko, vo, kp, vp, sc, dev(slots), 20, Hkv, D, block, dtype=KVC_F32, kv_dtype=kv_dtype)
    for x, b in ((k, ko), (v, vo)):
        x = x.astype(np.float64)
        s = np.abs(x).max(-1, keepdims=True) / TOP[kv_dtype]
        assert (np.abs(host(b, np.float32, x.shape) - x) <= half_step(x, s, kv_dtype) * 1.001).all()


