"""The operators around an 8-bit paged cache without a GPU: their refusals (validation precedes
any HIP call), the plan of a ragged batch, and the plain forms the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

from _cache8 import E4M3, chunk_attention, norm_rope, quantise, round_e4m3, values
from _helpers import tuning
from kvcache_amd import _native as N
from kvcache_amd import ops

P = 0x10000  # a 16-byte aligned address that the refused calls never touch


def refused(status, f, *a, **kw):
    with pytest.raises(N.KvcError) as e:
        f(*a, **kw)
    assert e.value.status == status, e.value
    return str(e.value)


def rope(**kw):
    a = dict(q=P, k_pool=2 * P, v_pool=3 * P, kv_scales=4 * P, qkv=5 * P, pos=P, slots=P, M=4, Hq=8, Hkv=2, D=64,
             BLOCK=16, theta=1e4)
    a.update(kw)
    return ops.qk_norm_rope_write(**a)


@pytest.mark.parametrize("kw", [dict(Hq=7), dict(Hkv=0), dict(M=-1), dict(BLOCK=0), dict(theta=1.0), dict(theta=np.inf),
                                dict(eps=-1.0), dict(eps=np.nan), dict(row_stride=8 * 64), dict(row_stride=12 * 64 + 4),
                                dict(kv_dtype=9), dict(kv_scales=None), dict(kv_scales=4 * P + 4), dict(q=P + 2),
                                dict(qkv=P), dict(qkv=None), dict(pos=None), dict(slots=None), dict(v_pool=None),
                                dict(k_pool=P + 8), dict(q_norm=P + 8), dict(k_norm=P + 2)])
def test_norm_rope_write_refuses(kw):
    refused(N.KVC_ERR_ARG, rope, **kw)


@pytest.mark.parametrize("kw", [dict(D=48), dict(D=512), dict(kv_dtype=N.KVC_F32), dict(Hq=1 << 17, Hkv=1 << 16, M=1)])
def test_norm_rope_write_unsupported(kw):
    refused(N.KVC_ERR_UNSUPPORTED, rope, **kw)


def write(**kw):
    a = dict(k=P, v=P, k_pool=P, v_pool=P, kv_scales=P, slot_map=P, rows=4, Hkv=2, D=64, BLOCK=16)
    a.update(kw)
    return ops.write_kv_q8(**a)


def read(**kw):
    a = dict(k=P, v=P, k_pool=P, v_pool=P, kv_scales=P, slot_map=P, rows=4, Hkv=2, D=64, BLOCK=16)
    a.update(kw)
    return ops.read_kv(**a)


@pytest.mark.parametrize("f", [write, read])
def test_write_and_read_refuse(f):
    for kw in (dict(rows=-1), dict(Hkv=0), dict(BLOCK=0), dict(dtype=N.KVC_I8), dict(kv_dtype=7), dict(kv_scales=None),
               dict(kv_scales=P + 4), dict(k=None), dict(v=P + 2), dict(k_pool=None), dict(v_pool=P + 8),
               dict(slot_map=None)):
        refused(N.KVC_ERR_ARG, f, **kw)
    for kw in (dict(D=96), dict(kv_dtype=N.KVC_F32), dict(rows=1 << 30)):
        refused(N.KVC_ERR_UNSUPPORTED, f, **kw)
    assert "kvc_write_kv_slots" in refused(N.KVC_ERR_UNSUPPORTED, write, kv_dtype=N.KVC_F16)


def attn(**kw):
    a = dict(q=P, out=P, k_pool=P, v_pool=P, kv_scales=P, table_all=P, table_len=9, work_dev=P, n_units=3, n_tiles=0,
             ws_rows=(0, 0), rows=4, Hq=8, Hkv=2, D=64, BLOCK=16, scale=0.125)
    a.update(kw)
    return ops.paged_chunk_attn(**a)


@pytest.mark.parametrize("kw", [dict(Hq=9), dict(Hkv=0), dict(BLOCK=0), dict(window=-1), dict(kv_dtype=5), dict(rows=-1),
                                dict(n_units=-1), dict(n_tiles=-1), dict(ws_rows=(-1, 0)), dict(ws_rows=(0, -1)), dict(n_tiles=1), dict(scale=np.nan),
                                dict(softcap=-1.0), dict(softcap=np.inf), dict(scale=3e38), dict(softcap=1e-38, scale=100.0), dict(q=None), dict(out=P + 2),
                                dict(k_pool=None), dict(v_pool=P + 8), dict(kv_scales=None), dict(kv_scales=P + 4),
                                dict(table_all=None), dict(table_len=0), dict(work_dev=None),
                                dict(ws_rows=(9, 0), workspace=(P + 4, 1 << 20))])
def test_chunk_attention_refuses(kw):
    refused(N.KVC_ERR_ARG, attn, **kw)


def test_chunk_attention_unsupported_and_workspace():
    refused(N.KVC_ERR_UNSUPPORTED, attn, D=80)
    refused(N.KVC_ERR_UNSUPPORTED, attn, kv_dtype=N.KVC_F32)
    refused(N.KVC_ERR_UNSUPPORTED, attn, n_units=1 << 30, Hkv=8)
    refused(N.KVC_ERR_UNSUPPORTED, attn, softcap=513.0)
    need = ops.chunk_workspace_size(8, 2, 64, (100, 50))
    assert need >= 2 * 100 * (64 + 2) * 4 + 2 * 50 * 2 * 64 * 2 and ops.chunk_workspace_size(8, 2, 64, (0, 0)) == 0
    refused(N.KVC_ERR_WORKSPACE, attn, ws_rows=(100, 50), workspace=(P, need - 1))


def test_nothing_to_do_is_no_call():
    attn(rows=0, q=None, out=None)
    attn(n_units=1, work_dev=None)  # a list that holds its header alone
    write(rows=0, k=None, v=None, k_pool=None, v_pool=None, slot_map=None)
    read(rows=0, k=None, v=None, k_pool=None, v_pool=None, slot_map=None)
    rope(M=0, q=None, qkv=None, pos=None, slots=None, k_pool=None, v_pool=None)


def test_plan_refuses():
    for q, t in (([2], [1]), ([-1], [5]), ([1, 1], [3])):
        refused(N.KVC_ERR_ARG, ops.chunk_plan, q, t, 8, 2, 64, 16)
    refused(N.KVC_ERR_ARG, ops.chunk_plan, [1], [1], 8, 3, 64, 16)
    refused(N.KVC_ERR_ARG, ops.chunk_plan, [1], [1], 8, 2, 64, 16, window=-1)
    refused(N.KVC_ERR_ARG, ops.chunk_plan, [1], [1], 8, 2, 64, 16, tab_off=[-1, 4])
    refused(N.KVC_ERR_ARG, ops.chunk_plan, [1], [1], 8, 2, 64, 16, tab_off=[0])
    refused(N.KVC_ERR_UNSUPPORTED, ops.chunk_plan, [1], [1], 8, 2, 72, 16)
    refused(N.KVC_ERR_UNSUPPORTED, ops.chunk_plan, [0, 0], [2 ** 31 - 1] * 2, 8, 2, 64, 1)
    refused(N.KVC_ERR_UNSUPPORTED, ops.chunk_plan, [1], [17], 8, 2, 64, 16, tab_off=[2 ** 31 - 2, 2 ** 31 - 1])
    L = N.lib()
    import ctypes as C
    n = [C.c_int(0) for _ in range(4)]
    one = np.ones(1, np.int32)
    assert L.kvc_chunk_plan(one.ctypes.data, one.ctypes.data, None, 1, 8, 2, 64, 16, N.KVC_I8, 0, one.ctypes.data, 1,
                            *map(C.byref, n)) == N.KVC_ERR_ARG  # capacity below the list
    assert L.kvc_chunk_plan(None, None, None, 1, 8, 2, 64, 16, N.KVC_I8, 0, None, 0, *map(C.byref, n)) == N.KVC_ERR_ARG
    assert L.kvc_chunk_plan(one.ctypes.data, one.ctypes.data, None, 1, 8, 2, 64, 16, N.KVC_I8, 0, None, 0, None,
                            *map(C.byref, n[1:])) == N.KVC_ERR_ARG


@pytest.mark.parametrize("Hq,Hkv,D,block", [(14, 2, 64, 16), (8, 8, 64, 16), (32, 8, 128, 16), (64, 2, 128, 32),
                                            (40, 1, 128, 16), (4, 2, 32, 16), (6, 3, 64, 10), (16, 2, 256, 64)])
@pytest.mark.parametrize("window", [0, 1, 100, 1000])
@pytest.mark.parametrize("tiles", [-1, 0, 1])
def test_plan_covers_every_row_and_key_once(Hq, Hkv, D, block, window, tiles):
    """Every (row, head) lies in units whose key ranges are disjoint and hold every key it sees;
    partial rows are disjoint and within n_records; ranges begin at whole 16-row subtiles."""
    rng = np.random.default_rng(Hq + window)
    group = Hq // Hkv
    for n, qmax, tmax in ((1, 1, 40000), (7, 1, 3000), (40, 90, 2000), (3, 2500, 9000), (200, 1, 900)):
        ql = rng.integers(0 if n > 1 else 1, qmax + 1, n)
        tl = ql + rng.integers(0, tmax, n)
        off = np.concatenate([[0], np.cumsum(-(-tl // block))]) + 5
        with tuning("chunk_tiles", tiles):
            work, nu, nt, (nr, nw) = ops.chunk_plan(ql, tl, Hq, Hkv, D, block, window=window, tab_off=off)
        assert (tiles != 0 or nt == 0) and (tiles != 1 or qmax <= 16 or D not in (64, 128) or block % 16 or nt > 0)
        assert work.shape == (nu, 16) and work[0, 0] == nu and work[0, 1] == nt and work[0, 2] == nr
        start = np.concatenate([[0], np.cumsum(ql)])
        covered = np.zeros((int(ql.sum()), group), np.int64)
        used = np.zeros(nr, bool)
        spans, widened = {}, {}
        tiles = 0
        for e in work[1:]:
            kind, row, tok, pos, h0, hn, j0, j1, c, nc, rec, tab, wide, wkey, w0, w1 = (int(x) for x in e)
            tiles += kind == 1
            s = int(np.searchsorted(start, row, side="right") - 1)
            assert start[s] <= row and row + tok <= start[s + 1] and pos == tl[s] - ql[s] + row - start[s]
            assert tab == off[s] and 0 <= h0 and h0 + hn <= group and 0 <= c < nc
            assert j0 % 16 == 0 and j0 < j1 <= pos + tok
            first = max(0, pos - window + 1) if window else 0
            spans.setdefault((row, tok, h0, hn), ([], first))[0].append((j0, j1))
            covered[row:row + tok, h0:h0 + hn] += j1 - j0
            if nc > 1:
                r = slice(rec + c * tok * hn, rec + (c + 1) * tok * hn)
                assert r.stop <= nr and not used[r].any()
                used[r] = True
            if kind == 1:  # its keys lie in the workspace, and it widens its share of them
                assert wide >= 0 and wkey <= j0 and wide + j1 - wkey <= nw and wkey <= w0 <= w1
                widened.setdefault((s, wide, wkey), []).append((w0, w1))
        assert tiles == nt and used.all() and (work[1:nt + 1, 0] == 1).all()
        rows = np.zeros(nw, np.int64)
        for (s, wide, wkey), shares in widened.items():
            for w0, w1 in shares:
                rows[wide + w0 - wkey:wide + w1 - wkey] += 1
            assert max(w1 for _, w1 in shares) == tl[s]
        assert (rows == 1).all()
        for (row, tok, h0, hn), (ranges, first) in spans.items():
            ranges.sort()
            assert ranges[0][0] <= first and all(a[1] == b[0] for a, b in zip(ranges, ranges[1:]))
            s = int(np.searchsorted(start, row, side="right") - 1)
            assert ranges[-1][1] == tl[s] - ql[s] + row - start[s] + tok
        assert (covered > 0).all()


def test_tile_knob():
    L = N.lib()
    v = C.c_int(7)
    assert L.kvc_get_tuning(b"chunk_tiles", C.byref(v)) == N.KVC_OK and v.value == -1
    for bad in (-2, 2):
        assert L.kvc_set_tuning(b"chunk_tiles", bad) == N.KVC_ERR_ARG


def test_plan_larger_than_its_first_buffer():
    """The binding's second call: many more units than four a sequence."""
    work, nu, nt, (nr, nw) = ops.chunk_plan([3000], [3000], 14, 2, 64, 10)
    assert nu > 68 and work.shape == (nu, 16) and work[0, 0] == nu and (work[1:, 2] > 0).all()
    n = [C.c_int(0) for _ in range(4)]
    q = np.array([3000], np.int32)
    small = np.zeros((4, 16), np.int32)
    assert N.lib().kvc_chunk_plan(q.ctypes.data, q.ctypes.data, None, 1, 14, 2, 64, 10, N.KVC_I8, 0, small.ctypes.data, 4,
                                  *map(C.byref, n)) == N.KVC_ERR_ARG
    assert n[0].value == nu and (small == 0).all()


def test_plan_of_an_empty_batch():
    for q, t in (([], []), ([0, 0], [0, 30])):
        work, nu, nt, rows = ops.chunk_plan(q, t, 8, 2, 64, 16)
        assert (nu, nt, rows) == (1, 0, (0, 0)) and work[0, 0] == 1


def test_plain_forms():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 3, 64))
    for kv, tol in ((N.KVC_I8, 0.5 / 127), (N.KVC_E4M3, 2.0 ** -4)):
        c, s = quantise(x, kv)
        assert (np.abs(values(c, kv) * s[..., None] - x) <= tol * np.abs(x).max(-1, keepdims=True) * 1.001).all()
    assert E4M3[0x7E] == 448 and E4M3[1] == 2.0 ** -9 and np.isnan(E4M3[0x7F]) and E4M3[0xB8] == -1
    assert (round_e4m3(np.array([17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10])) == [16, 20, 0, 2.0 ** -8]).all()
    q, k, v = (rng.standard_normal(s) for s in ((4, 6, 64), (9, 2, 64), (9, 2, 64)))
    out, mag, _ = chunk_attention(q, k, v, 4, 3, 2.0, 0.1)
    z = np.einsum("ihd,jhd->hij", q, np.repeat(k, 3, 1)) * 0.1
    z = 2 * np.tanh(z / 2)
    p, j = 5 + np.arange(4)[:, None], np.arange(9)[None]
    z = np.where((j <= p) & (j > p - 3), z, -np.inf)
    e = np.exp(z - z.max(-1, keepdims=True))
    e /= e.sum(-1, keepdims=True)
    assert np.abs(np.einsum("hij,jhd->ihd", e, np.repeat(v, 3, 1)) - out).max() < 1e-12 and (mag >= np.abs(out)).all()
    y, _ = norm_rope(x, None, 0.0, np.zeros(5), 1e4)
    assert (y == x).all()
    y, _ = norm_rope(x, np.ones(64), 0.0, np.array([0, 3, 9, 100, 10 ** 6]), 1e4)
    assert np.abs((y ** 2).mean(-1) - 1).max() < 1e-12  # a rotation keeps the norm
