"""Attention of a ragged batch of chunks over a paged cache (fp16, int8, e4m3) against a plain
64-bit form of the same dequantised cache."""
import ctypes as C

import numpy as np
import pytest

from _cache8 import (NAME, chunk_attention, chunk_bound, code_dtype, norm_rope, quantise, values)
from _helpers import dev, host, say, tuning
from kvcache_amd import KVC_E4M3, KVC_F16, KVC_I8, ops
from kvcache_amd._native import check, lib
from kvcache_amd.device import DeviceBuffer, Stream, synchronize

pytestmark = pytest.mark.gpu
ALL = [KVC_F16, KVC_I8, KVC_E4M3]


@pytest.fixture(params=[-1, 1], ids=["auto", "tiles"], autouse=True)
def tiles(request):
    """Batches this small go to units of 16 rows by themselves; each test runs with tiles as well."""
    with tuning("chunk_tiles", request.param):
        yield request.param


class Batch:
    """A ragged batch over a paged cache: the last block's unused rows, and blocks that no table
    names, hold NaN (fp16, e4m3) or extreme codes with NaN scales."""

    def __init__(self, q_lens, kv_lens, Hq, Hkv, D, block, kv_dtype, seed=0, spread=0.5, k_std=1.0, spare=3):
        rng = np.random.default_rng(seed)
        self.ql, self.tl = np.asarray(q_lens, np.int32), np.asarray(kv_lens, np.int32)
        self.Hq, self.Hkv, self.D, self.block, self.kv = Hq, Hkv, D, block, kv_dtype
        nblk = -(-self.tl // block)
        self.off = np.concatenate([[0], np.cumsum(nblk)]).astype(np.int32)
        nb = int(self.off[-1]) + spare
        self.table = rng.permutation(nb)[: max(int(self.off[-1]), 1)].astype(np.int32)
        self.rows = int(self.ql.sum())
        self.q = rng.standard_normal((self.rows, Hq, D)).astype(np.float16)
        shape = (nb, Hkv, block, D)
        bad = {KVC_F16: np.nan, KVC_I8: -128, KVC_E4M3: 0x7F}[kv_dtype]
        self.pools = [np.full(shape, bad, code_dtype(kv_dtype)) for _ in "kv"]
        self.scales = np.full(shape[:3] + (2,), np.nan, np.float32)
        self.tok = [[], []]  # dequantised K, V [t, Hkv, D] of each sequence
        for s, t in enumerate(self.tl):
            at = np.arange(t)
            blk, pos = self.table[self.off[s] + at // block], at % block
            for i in (0, 1):
                x = rng.standard_normal((t, Hkv, D)) * np.exp(spread * rng.standard_normal((t, Hkv, 1)))
                x = x * (k_std if i == 0 else 1.0)
                if kv_dtype == KVC_F16:
                    x = x.astype(np.float16)
                    self.pools[i][blk, :, pos] = x
                    self.tok[i].append(x.astype(np.float64))
                else:
                    c, sc = quantise(x, kv_dtype)
                    self.pools[i][blk, :, pos], self.scales[blk, :, pos, i] = c, sc
                    self.tok[i].append(values(c, kv_dtype) * sc[..., None].astype(np.float64))

    def run(self, scale=None, window=0, cap=0.0, workspace="own", stream=None, tab_off=True):
        D = self.D
        scale = D ** -0.5 if scale is None else scale
        work, nu, nt, nr = ops.chunk_plan(self.ql, self.tl, self.Hq, self.Hkv, D, self.block, kv_dtype=self.kv,
                                          window=window, tab_off=self.off if tab_off else None)
        self.plan = (work, nu, nt, nr)
        out = dev(np.full((self.rows + 2, self.Hq, D), 7, np.float16))
        ws = None
        if workspace == "own":
            size = ops.chunk_workspace_size(self.Hq, self.Hkv, D, nr)
            ws = dev(np.full(max(size, 16) // 4, np.nan, np.float32))
        self.bufs = [dev(self.q), dev(self.pools[0]), dev(self.pools[1]), dev(self.scales), dev(self.table), dev(work)]
        q, k, v, sc, tab, w = self.bufs
        say(f"chunk attention {NAME[self.kv]} N={len(self.ql)} rows={self.rows} Hq={self.Hq} Hkv={self.Hkv} D={D} "
            f"block={self.block} window={window} cap={cap} units={nu} tiles={nt} workspace rows={nr}")
        ops.paged_chunk_attn(q, out, k, v, None if self.kv == KVC_F16 else sc, tab, len(self.table), w, nu, nt, nr,
                             self.rows, self.Hq, self.Hkv, D, self.block, scale, kv_dtype=self.kv, softcap=cap,
                             window=window, workspace=ws, stream=stream)
        synchronize()
        got = host(out, np.float16, (self.rows + 2, self.Hq, D))
        assert (got[self.rows:] == 7).all()  # rows behind the last sequence
        return got[: self.rows].astype(np.float64)

    def want(self, scale=None, window=0, cap=0.0):
        scale = self.D ** -0.5 if scale is None else scale
        parts, row = [], 0
        for s, n in enumerate(self.ql):
            parts.append(chunk_attention(self.q[row:row + n], self.tok[0][s], self.tok[1][s], n, window, cap, scale))
            row += n
        return [np.concatenate([p[i] for p in parts]) for i in range(3)]

    def check(self, **kw):
        run_kw = {k: kw.pop(k) for k in ("workspace", "stream", "tab_off") if k in kw}
        got = self.run(**kw, **run_kw)
        out, mag, big = self.want(**kw)
        bound = chunk_bound(out, mag, big, self.D, kw.get("cap", 0.0), kv16=self.kv != KVC_F16)
        err = np.abs(got - out)
        assert (err <= bound).all(), (float((err / bound).max()), np.unravel_index((err / bound).argmax(), err.shape))
        return got


SHAPES = [  # q_lens, kv_lens, Hq, Hkv, D, block
    ([1], [1], 8, 8, 64, 16),                                  # one token that sees itself
    ([1, 1, 1], [1, 17, 300], 14, 2, 64, 16),
    ([1] * 9, [5, 33, 64, 65, 128, 129, 500, 1000, 2100], 32, 8, 128, 16),
    ([3, 0, 1, 40], [3, 20, 90, 100], 14, 2, 64, 16),          # a sequence without new tokens
    ([130], [130], 8, 2, 128, 16),                             # a prompt from its start
    ([70, 1, 5], [700, 2500, 6], 16, 4, 128, 32),
    ([257], [1200], 6, 6, 64, 64),
    ([1, 2], [4000, 4001], 3, 1, 64, 16),
    ([2, 1], [40, 70], 64, 2, 64, 16),                         # 32 heads for each KV head
    ([5, 1], [37, 130], 40, 1, 128, 16),                       # 40: more than a row tile
    ([33], [95], 5, 5, 128, 128),
]
OTHER = [  # head_dims and blocks outside the matrix-core kernels
    ([1, 9, 2], [1, 30, 150], 4, 2, 32, 16),
    ([1, 20], [200, 60], 8, 2, 256, 16),
    ([4, 1], [50, 77], 6, 3, 64, 10),
    ([1, 7], [23, 40], 4, 1, 128, 1),
    ([12], [1300], 2, 1, 128, 48),
]


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
@pytest.mark.parametrize("shape", SHAPES + OTHER, ids=lambda s: f"{len(s[0])}x{max(s[0])}-{s[2]}q{s[3]}kv-d{s[4]}-b{s[5]}")
def test_against_64_bits(shape, kv):
    Batch(*shape, kv).check()


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
@pytest.mark.parametrize("window", [1, 16, 33, 200, 5000])
def test_window(window, kv):
    Batch([90, 1, 1, 6], [400, 700, 3, 250], 8, 2, 64, 16, kv, seed=window).check(window=window)
    Batch([40, 1], [300, 130], 8, 8, 128, 16, kv, seed=window).check(window=window, cap=15.0)


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
@pytest.mark.parametrize("cap,std", [(30.0, 1.0), (5.0, 6.0), (50.0, 30.0), (512.0, 1.0), (0.05, 1.0)])
def test_softcap(cap, std, kv):
    Batch([70, 1, 3], [200, 333, 64], 14, 2, 64, 16, kv, k_std=std).check(cap=cap)
    Batch([5, 20], [40, 21], 4, 4, 32, 16, kv, k_std=std).check(cap=cap, scale=-0.2)


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
@pytest.mark.parametrize("D", [64, 128])
def test_large_scores_and_values_of_many_sizes(D, kv):
    """One key decides a row; rows of V whose sizes differ by up to e^8."""
    Batch([80, 1], [333, 900], 8, 2, D, 16, kv, seed=3, k_std=25.0).check()
    Batch([80, 1], [333, 900], 8, 2, D, 16, kv, seed=4, spread=2.0, k_std=0.3).check()
    Batch([80, 1], [333, 900], 8, 2, D, 16, kv, seed=5).check(scale=-0.1)
    Batch([80, 1], [333, 900], 8, 2, D, 16, kv, seed=6).check(scale=0.0)
    Batch([80, 1], [333, 900], 8, 2, D, 16, kv, seed=7, spread=0.1, k_std=9000.0).check(scale=40.0)  # (K up to 6e4)
    Batch([80, 1], [333, 900], 8, 2, D, 16, kv, seed=8, k_std=1e-4).check(scale=1000.0)


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
@pytest.mark.parametrize("D,hq,hkv", [(64, 14, 2), (128, 8, 2), (128, 2, 2)])
def test_many_rows_over_split_keys(D, hq, hkv, kv, tiles):
    """Few tiles over many keys: their key ranges are split and merged, with whole tiles beside them;
    a window that leaves chunks of some rows empty; a first token that sees a single key."""
    b = Batch([140, 66, 3], [5000, 66, 3000], hq, hkv, D, 16, kv, seed=60)
    a = b.check()
    work, nu, nt, (nr, nw) = b.plan
    if tiles == 1:
        assert nt > 0 and nr > 0 and (kv == KVC_F16) == (nw == 0)
        kinds = np.asarray(work).reshape(-1, 16)[1:]
        assert len(kinds) == nu - 1
    assert (b.run() == a).all()
    Batch([140, 66, 3], [5000, 66, 3000], hq, hkv, D, 16, kv, seed=61).check(window=2100, cap=20.0)


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
@pytest.mark.parametrize("D", [32, 64, 128])
def test_what_is_not_finite_stays_with_the_rows_that_see_it(D, kv):
    """A V row of Inf or NaN at key j reaches rows from position j on, and up to j + window - 1."""
    for window in (0, 20):
        b = Batch([60, 1, 3], [75, 75, 75], 4, 2, D, 16, kv, seed=7)
        hit = {0: 40, 2: 73}  # sequence -> key
        for s, j in hit.items():
            blk, at = b.table[b.off[s] + j // 16], j % 16
            if kv == KVC_F16:
                b.pools[1][blk, 0, at, 5] = np.inf if s else np.nan
            else:
                b.scales[blk, 0, at, 1] = np.nan
        got = b.run(window=window)
        clean = Batch([60, 1, 3], [75, 75, 75], 4, 2, D, 16, kv, seed=7)
        ok = clean.run(window=window)
        row = 0
        for s, n in enumerate(b.ql):
            for i in range(n):
                p = b.tl[s] - n + i
                sees = s in hit and hit[s] <= p and (not window or hit[s] > p - window)
                g = got[row + i]
                assert np.isfinite(g[2:]).all()                     # the other KV head's
                if not sees:
                    assert (g == ok[row + i]).all(), (window, s, i)
                elif kv == KVC_F16:
                    assert not np.isfinite(g[:2, 5]).any() and np.isfinite(np.delete(g[:2], 5, 1)).all()
                else:
                    assert np.isnan(g[:2]).all()
            row += n


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
def test_a_key_that_is_nan_reaches_the_rows_that_see_it(kv):
    b = Batch([50, 1], [50, 90], 4, 2, 64, 16, kv, seed=8)
    j = 31
    blk, at = b.table[b.off[0] + j // 16], j % 16
    if kv == KVC_F16:
        b.pools[0][blk, 1, at, 0] = np.nan
    else:
        b.scales[blk, 1, at, 0] = np.nan
    got = b.run()
    assert np.isfinite(got[:, :2]).all() and np.isfinite(got[:j]).all() and np.isfinite(got[50:]).all()
    assert np.isnan(got[j:50, 2:]).all()


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
def test_workspaces_streams_and_repeats(kv):
    """A library-owned workspace, a caller's, another stream and a second run: the same bits."""
    b = Batch([1, 4, 1], [5000, 3000, 200], 8, 2, 128, 16, kv, seed=9)
    a = b.check()
    st = Stream()
    for kw in ({"workspace": None}, {"stream": st.handle}, {"tab_off": False}, {}):
        assert (b.run(**kw) == a).all()
    assert b.plan[3][0] > 0


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
def test_two_streams_at_once(kv):
    """Two batches in flight on streams of their own, each on its library-owned workspace."""
    bs = [Batch([1, 3], [6000, 2000 + 500 * i], 8, 2, 64, 16, kv, seed=20 + i) for i in range(2)]
    want = [b.run() for b in bs]
    sts = [Stream(), Stream()]
    outs = []
    for _ in range(3):
        for b, st in zip(bs, sts):
            q, k, v, sc, tab, w = b.bufs
            out = dev(np.zeros((b.rows, 8, 64), np.float16))
            _, nu, nt, nr = b.plan
            ops.paged_chunk_attn(q, out, k, v, None if kv == KVC_F16 else sc, tab, len(b.table), w, nu, nt, nr, b.rows,
                                 8, 2, 64, 16, 0.125, kv_dtype=kv, stream=st.handle)
            outs.append(out)
    synchronize()
    for i, o in enumerate(outs):
        assert (host(o, np.float16, (bs[i % 2].rows, 8, 64)) == want[i % 2]).all()


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
@pytest.mark.parametrize("D", [64, 128])
def test_captured_launch_replays_other_plans(D, kv):
    """One captured launch serves every step: plan, table, q and cache change in place between replays."""
    Hq, Hkv, block = 8, 2, 16
    steps = [Batch([1, 70, 1], [3000, 90, 40], Hq, Hkv, D, block, kv, seed=30, spare=40),
             Batch([1, 1], [700, 1500], Hq, Hkv, D, block, kv, seed=31, spare=40),
             Batch([60, 1, 1, 1], [1500, 20, 2, 1000], Hq, Hkv, D, block, kv, seed=32, spare=40)]
    want = [b.run() for b in steps]
    tiles = max(b.plan[2] for b in steps)
    cap = [max(b.plan[1] - b.plan[2] for b in steps) + tiles, tiles,
           tuple(max(b.plan[3][i] for b in steps) for i in (0, 1))]
    rows = max(b.rows for b in steps)
    size = [max(getattr(b, a).nbytes for b in steps) for a in ("q", "scales", "table")]
    pool = max(b.pools[0].nbytes for b in steps)
    q, sc, tab = (DeviceBuffer(s) for s in size)
    kp, vp, work = DeviceBuffer(pool), DeviceBuffer(pool), DeviceBuffer(cap[0] * 64)
    out = dev(np.zeros((rows, Hq, D), np.float16))
    wss = ops.chunk_workspace_size(Hq, Hkv, D, cap[2])
    ws = dev(np.full(max(wss, 16) // 4, np.nan, np.float32))
    st = Stream()
    L = lib()
    ex = C.c_void_p()
    ntab = max(len(b.table) for b in steps)
    check(L.kvc_graph_begin(st.handle))
    ops.paged_chunk_attn(q, out, kp, vp, None if kv == KVC_F16 else sc, tab, ntab, work, *cap, rows, Hq, Hkv, D, block,
                         D ** -0.5, kv_dtype=kv, workspace=ws, stream=st.handle)
    check(L.kvc_graph_end(st.handle, C.byref(ex)))
    for i in (0, 1, 2, 1, 0):
        b = steps[i]
        for buf, a in ((q, b.q), (sc, b.scales), (tab, b.table), (kp, b.pools[0]), (vp, b.pools[1]), (work, b.plan[0])):
            buf.upload(a)
        out.upload(np.full((rows, Hq, D), 3, np.float16))
        check(L.kvc_graph_launch(ex, st.handle))
        st.synchronize()
        got = host(out, np.float16, (rows, Hq, D)).astype(np.float64)
        bound = 2.0 ** -10 * np.abs(want[i]) + 2.0 ** -12  # (captured for more splits: the same plan, the same bits)
        assert (np.abs(got[: b.rows] - want[i]) <= bound).all() and (got[b.rows:] == 3).all()
        assert (got[: b.rows] == want[i]).all()
    check(L.kvc_graph_destroy(ex))


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
def test_two_captured_launches_share_a_workspace(kv):
    """Replayed in turn on one stream, with other contents in the workspace now and then."""
    bs = [Batch([1, 70, 2], [4000, 2500, 900], 8, 2, 64, 16, kv, seed=70), Batch([3, 1, 33], [900, 6000, 1500], 8, 2, 64, 16, kv, seed=71)]
    want = [b.run() for b in bs]
    assert all(b.plan[3][0] > 0 for b in bs)
    n = max(ops.chunk_workspace_size(8, 2, 64, b.plan[3]) for b in bs)
    ws, st, L = DeviceBuffer(n), Stream(), lib()
    graphs = []
    for b in bs:
        q, k, v, sc, tab, w = b.bufs
        out, ex = dev(np.zeros((b.rows, 8, 64), np.float16)), C.c_void_p()
        check(L.kvc_graph_begin(st.handle))
        ops.paged_chunk_attn(q, out, k, v, None if kv == KVC_F16 else sc, tab, len(b.table), w, *b.plan[1:], b.rows, 8, 2,
                             64, 16, 0.125, kv_dtype=kv, workspace=ws, stream=st.handle)
        check(L.kvc_graph_end(st.handle, C.byref(ex)))
        graphs.append((ex, out))
    rng = np.random.default_rng(0)
    for i in (0, 1, 1, 0, 0, 1):
        if i == 0:
            ws.upload(rng.integers(0, 256, n, dtype=np.uint8))
        ex, out = graphs[i]
        out.upload(np.zeros((bs[i].rows, 8, 64), np.float16))
        check(L.kvc_graph_launch(ex, st.handle))
        st.synchronize()
        assert (host(out, np.float16, want[i].shape) == want[i]).all()
    for ex, _ in graphs:
        check(L.kvc_graph_destroy(ex))


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
@pytest.mark.parametrize("D", [32, 64, 128])
def test_output_in_place_of_the_queries(D, kv):
    b = Batch([1, 70, 2], [3000, 90, 900], 8, 2, D, 16, kv, seed=72)
    want = b.run()
    q, k, v, sc, tab, w = b.bufs
    ops.paged_chunk_attn(q, q, k, v, None if kv == KVC_F16 else sc, tab, len(b.table), w, *b.plan[1:], b.rows, 8, 2, D, 16,
                         D ** -0.5, kv_dtype=kv)
    synchronize()
    assert (host(q, np.float16, want.shape) == want).all()


@pytest.mark.parametrize("D", [32, 64, 128])
def test_signed_scales(D):
    """Codes and scale of opposite sign stand for the same row."""
    b = Batch([1, 70], [700, 90], 8, 2, D, 16, KVC_I8, seed=73)
    for i in (0, 1):
        b.pools[i] = np.where(b.pools[i] == -128, b.pools[i], -b.pools[i]).astype(np.int8)
    b.scales = -b.scales
    b.check()


@pytest.mark.parametrize("kv", [KVC_I8, KVC_E4M3], ids=NAME.get)
def test_cache_past_32_bits(kv):
    """Pools of more than 2^32 bytes: blocks at their far end are found."""
    Hq, Hkv, D, block = 8, 8, 128, 16
    nb = (1 << 32) // (Hkv * D * block) + 40
    b = Batch([20, 1], [100, 300], Hq, Hkv, D, block, kv, seed=40)
    far = np.arange(nb - len(b.table), nb, dtype=np.int32)[::-1].copy()
    bufs = [DeviceBuffer(nb * Hkv * block * n) for n in (D, D, 8)]
    out = dev(np.zeros((b.rows, Hq, D), np.float16))
    want = b.run()
    row = Hkv * block
    for j, (src, dst) in enumerate(zip(b.table, far)):
        for buf, a, n in zip(bufs, (*b.pools, b.scales), (D, D, 8)):
            x = np.ascontiguousarray(a[src])
            check(lib().kvc_memcpy_h2d(buf.ptr + int(dst) * row * n, x.ctypes.data, x.nbytes, None))
    synchronize()
    work, nu, nt, nr = b.plan
    ws = DeviceBuffer(max(ops.chunk_workspace_size(Hq, Hkv, D, nr), 16))
    ops.paged_chunk_attn(b.bufs[0], out, *bufs, dev(far), len(far), dev(work), nu, nt, nr, b.rows, Hq, Hkv, D, block,
                         D ** -0.5, kv_dtype=kv, workspace=ws)
    synchronize()
    assert (host(out, np.float16, want.shape) == want).all()


@pytest.mark.parametrize("kv", ALL, ids=NAME.get)
def test_a_sequence_from_its_prompt_to_its_last_token(kv):
    """The operators as they are used: every step's q|k|v rows go through norm, rotary and cache
    write, then the chunk attends; chunks of a prompt first, then single tokens; two sequences."""
    Hq, Hkv, D, block, theta, eps = 8, 2, 64, 16, 1e4, 1e-6
    rng = np.random.default_rng(50)
    qn, kn = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float16) for _ in "qk")
    steps = [(33, 5), (20, 40), (1, 1), (1, 17), (1, 1)]
    total = np.sum(steps, 0)
    nblk = -(-total // block)
    off = np.concatenate([[0], np.cumsum(nblk)]).astype(np.int32)
    nb = int(off[-1]) + 1
    table = rng.permutation(nb)[: off[-1]].astype(np.int32)
    shape = (nb, Hkv, block, D)
    dk, dv = dev(np.zeros(shape, code_dtype(kv))), dev(np.zeros(shape, code_dtype(kv)))
    sc = dev(np.zeros(shape[:3] + (2,), np.float32))
    scp = None if kv == KVC_F16 else sc
    tab, dqn, dkn = dev(table), dev(qn), dev(kn)
    have = np.zeros(2, int)
    for step in steps:
        n = np.array(step)
        rows = int(n.sum())
        x = rng.standard_normal((rows, Hq + 2 * Hkv, D)).astype(np.float16)
        pos = np.concatenate([np.arange(have[s], have[s] + n[s]) for s in (0, 1)]).astype(np.int32)
        seq = np.repeat([0, 1], n)
        slots = (table[off[seq] + pos // block] * block + pos % block).astype(np.int32)
        have += n
        q, out = dev(np.zeros((rows, Hq, D), np.float16)), dev(np.zeros((rows, Hq, D), np.float16))
        say(f"step {step} {NAME[kv]}")
        ops.qk_norm_rope_write(q, dk, dv, scp, dev(x), dev(pos), dev(slots), rows, Hq, Hkv, D, block, theta, q_norm=dqn,
                               k_norm=dkn, eps=eps, kv_dtype=kv)
        work, nu, nt, nr = ops.chunk_plan(n, have, Hq, Hkv, D, block, kv_dtype=kv, tab_off=off)
        ops.paged_chunk_attn(q, out, dk, dv, scp, tab, len(table), dev(work), nu, nt, nr, rows, Hq, Hkv, D, block,
                             D ** -0.5, kv_dtype=kv)
        synchronize()
        got, qs = host(out, np.float16, (rows, Hq, D)), host(q, np.float16, (rows, Hq, D))
        ref, size = norm_rope(x[:, :Hq], qn, eps, pos, theta)
        assert np.abs(qs - ref).max() < 2e-2
        # the attention over what the cache holds (as read back), each row to its position
        at = np.concatenate([np.arange(t) for t in have])
        who = np.repeat([0, 1], have)
        rs = (table[off[who] + at // block] * block + at % block).astype(np.int32)
        kr, vr = (dev(np.zeros((len(rs), Hkv, D), np.float32)) for _ in "kv")
        ops.read_kv(kr, vr, dk, dv, scp, dev(rs), len(rs), Hkv, D, block, dtype=0, kv_dtype=kv)
        k, v = (host(b, np.float32, (len(rs), Hkv, D)).astype(np.float64) for b in (kr, vr))
        row = 0
        for s in (0, 1):
            out64, mag, big = chunk_attention(qs[row:row + n[s]], k[who == s], v[who == s], n[s], 0, 0.0, D ** -0.5)
            bound = chunk_bound(out64, mag, big, D, 0.0, kv16=kv != KVC_F16)
            assert (np.abs(got[row:row + n[s]] - out64) <= bound).all()
            row += n[s]
