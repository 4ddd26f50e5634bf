// chunk_attn.hip -- attention of a ragged batch of chunks over a paged cache: the host plan and
// the launches (kernels in chunk_attn.hpp).
#include "chunk_tile.hpp"

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

namespace kvc {
namespace {

constexpr size_t kPartAlign = 256;
size_t up(size_t x, size_t a) { return (x + a - 1) / a * a; }
size_t acc_bytes(int Hkv, int D, int n_records) { return up((size_t)Hkv * n_records * D * sizeof(float), kPartAlign); }
size_t wide_bytes(int Hkv, int D, int n_wide) { return up((size_t)Hkv * n_wide * D * 2, kPartAlign); }
size_t ml_bytes(int Hkv, int n_records) { return up((size_t)Hkv * n_records * 2 * sizeof(float), kPartAlign); }
size_t ctr_bytes(int Hkv, int n_records) { return up((size_t)Hkv * n_records * sizeof(unsigned long long), kPartAlign); }
size_t factor_bytes(int Hkv, int n_wide) { return up((size_t)Hkv * n_wide * sizeof(float), kPartAlign); }

int check_shape(int Hq, int Hkv, int D, int BLOCK, int kv_dtype, int window) {
    if (kv_dtype == KVC_F32) return set_error(KVC_ERR_UNSUPPORTED, "the cache must be KVC_F16, KVC_I8 or KVC_E4M3");
    if (kv_dtype != KVC_F16 && kv_dtype != KVC_I8 && kv_dtype != KVC_E4M3)
        return set_error(KVC_ERR_ARG, "kv_dtype must be KVC_F16, KVC_I8 or KVC_E4M3");
    if (Hq <= 0 || Hkv <= 0 || Hq % Hkv) return set_error(KVC_ERR_ARG, "Hq must be a positive multiple of Hkv");
    if (D != 32 && D != 64 && D != 128 && D != 256)
        return set_error(KVC_ERR_UNSUPPORTED, "head_dim must be 32, 64, 128 or 256");
    if (BLOCK <= 0 || window < 0) return set_error(KVC_ERR_ARG, "BLOCK must be > 0 and window >= 0");
    return KVC_OK;
}

// The matrix-core kernels: head_dim 64 or 128, and blocks that hold whole 16-row subtiles,
// found by a shift.
bool matrix_path(int D, int BLOCK) { return (D == 64 || D == 128) && BLOCK >= 16 && (BLOCK & (BLOCK - 1)) == 0; }

// One tile of rows before its key range is cut.
struct Tile {
    int kind, row0, ntok, pos0, h0, hn, j0, j1, tab;
    int wide, wkey;  // 8-bit caches: the workspace row of key wkey
};

struct PlanUnit {
    int f[kChunkInts];
    long long cost;
};

// Chunks of `len` keys at a target of c (up to 1.5 c stay whole).
int chunks_of(long long len, long long c) { return len > c * 3 / 2 ? (int)((len + c - 1) / c) : 1; }

// Keys per chunk of the units of 16 rows, `keys` of them over all units and KV heads.  A batch is cut
// for one workgroup a CU (256) down to 256 keys (one round of four waves), for two down to 1024.
// int8, 32q/8kv, D 128: one sequence of 4000 38.4 us whole, 15.2 in chunks of 1024, 10.7 in 256; 64 of
// 32..4096 33.7 for 256 workgroups, 27.9 in chunks of 1024, 30.6 of 512; 128 of 16..2048 (8q/8kv, D 64,
// e4m3) 16.4, 15.1 and 16.8; 48 of 32..4096, 1 to 300 tokens (14q/2kv, D 64) 21.8, 17.1 and 16.9.
// At most 32 chunks of a sequence, whose arrivals are served one after the other (one of 20000,
// 8q/8kv: 12.3 us in 32 chunks, 13.4 in 24, 17.8 in 40).
// A few workgroups more than the card holds at once (D 128: 512) are a round of their own where all are
// about as long: then longer chunks that fit are taken (24 of 4000, 32q/8kv, D 128, int8: 57.0 -> 49.1
// us, of 1000..8000 48.8 -> 39.5; at D 64, three workgroups a CU, it gained nothing).
long long stream_chunk(const std::vector<Tile>& tiles, int Hkv, int D) {
    long long keys = 0, longest = 0;
    for (const Tile& t : tiles) {
        if (t.kind == kKindTile) continue;
        keys += t.j1 - t.j0;
        longest = std::max<long long>(longest, t.j1 - t.j0);
    }
    keys *= Hkv;
    const long long one = (keys + 255) / 256, two = (keys + 511) / 512;
    long long c = std::max(256LL, std::min(one, std::max(two, 1024LL)));
    c = (std::max<long long>(c, (longest + 31) / 32) + 63) / 64 * 64;
    auto units = [&](long long size) {
        long long u = 0;
        for (const Tile& t : tiles)
            if (t.kind != kKindTile) u += chunks_of(t.j1 - t.j0, size);
        return u * Hkv;
    };
    const long long n = units(c);
    if (D == 128 && c < longest && n > 512 && n <= 640 && 4 * keys >= 3 * n * c)
        for (long long size = c + 64; size <= 2 * c; size += 64)
            if (units(size) <= 512) return size;
    return c;
}

// Keys per chunk of the tiles (INT_MAX: whole): the shortest estimate among whole tiles and chunks
// for one, two or three rounds of the card's workgroups.  A set of 64 keys takes a tile of 256 rows
// 2.1 us at head_dim 128 (one workgroup a CU), 1.8 at 64 (two a CU), a unit another 4; the partials
// are written and read at about 4 TB/s and merged by a launch of 4 us.  2000 tokens of 32 heads
// behind 4000, D 128 (256 workgroups whole): 103 us whole, 125 in 320 workgroups.  At least 512 keys
// (D 128: 256): 700 behind 3000, 14q/2kv, D 64, int8, 34 us in chunks of 512, 39 of 256; 400 behind
// 1000, 32q/8kv, D 128, 37.5 and 35.6.
long long tile_chunk(const std::vector<Tile>& tiles, int Hkv, int D) {
    long long keys = 0, longest = 0, rows_keys = 0, n = 0;
    for (const Tile& t : tiles) {
        if (t.kind != kKindTile) continue;
        const long long len = t.j1 - t.j0;
        keys += len;
        longest = std::max(longest, len);
        rows_keys += t.ntok * t.hn;
        ++n;
    }
    if (n == 0) return INT_MAX;
    const double per_key = (D == 128 ? 2.1 : 1.8) / 64, unit = 4.0;
    const long long slots = D == 128 ? 256 : 512;
    auto units = [&](long long c) {
        long long u = 0;
        for (const Tile& t : tiles)
            if (t.kind == kKindTile) u += chunks_of(t.j1 - t.j0, c);
        return u * Hkv;
    };
    auto estimate = [&](long long c) {
        const long long u = units(c);
        const double mean = (double)keys * Hkv / u, top = (double)std::min(longest, c * 3 / 2);
        const double rounds = (double)((u + slots - 1) / slots);
        double t = u <= slots ? unit + per_key * top
                              : std::min(rounds * (unit + per_key * top),
                                         std::max(rounds * (unit + per_key * mean), (u * unit + per_key * keys * Hkv) / slots +
                                                                                        0.4 * (unit + per_key * top)));
        if (u > n * Hkv) t += 4.0 + 8.0 * rows_keys * Hkv * D * ((double)u / (n * Hkv)) / 4e6;
        return t;
    };
    long long best = INT_MAX;
    double least = estimate(INT_MAX / 2);
    for (int k = 1; k <= 3; ++k) {
        long long c = std::max(D == 128 ? 256LL : 512LL, (keys * Hkv + k * slots - 1) / (k * slots));
        for (int i = 0; i < 40 && c < longest && units(c) > k * slots; ++i) c += c / 16 + 1;
        c = (c + 63) / 64 * 64;
        if (c >= longest) continue;
        const double t = estimate(c);
        if (t < 0.97 * least) least = t, best = c;
    }
    return best;
}

// The batch as units.  Where the sequences of more than kTileRows rows (token, head) of a KV head
// make enough work, they are cut into tiles of up to 256 rows; all else into units of 16.
constexpr int kTileRows = 64;
void plan_units(const int* q_lens, const int* kv_lens, const int* tab_off, int N, int Hq, int Hkv, int D, int BLOCK,
                int kv_dtype, int window, std::vector<PlanUnit>& units, long long& records, long long& wide) {
    const int group = Hq / Hkv;
    auto first_key = [&](int pos) { return window > 0 ? std::max(0, pos - window + 1) / 64 * 64 : 0; };
    // Tiles reach about three times the rate of units of 16 rows, but take a launch or two more (merge;
    // 8-bit caches: widening).  One sequence, int8 (fp16), units of 16 and tiles: 14q/2kv, D 64, 400
    // tokens behind 1000 (1.7 GFLOP) 16 and 25 us (12 and 20), 1000 behind 1000 (5.4) 30 and 30 (28 and
    // 24), 400 behind 4000 (6.0) 40 and 31 (29 and 24); 32q/8kv, D 128, 64 behind 4000 (4.2) 24 and 33
    // (23 and 25), 500 behind 500 (6.1) 31 and 34 (27 and 27), 400 behind 1000 (7.9) 38 and 36 (35 and
    // 29), 150 behind 4000 (10) 51 and 41 (49 and 32).
    bool tiled = false;
    if (matrix_path(D, BLOCK)) {
        double flops = 0;
        for (int s = 0; s < N; ++s)
            if ((long long)q_lens[s] * group > kTileRows) {
                const double n = q_lens[s], seen = kv_lens[s] - n + 0.5 * (n + 1);
                flops += 4.0 * D * Hq * n * (window > 0 ? std::min<double>(seen, window) : seen);
            }
        const int knob = tuning().chunk_tiles;
        tiled = knob >= 0 ? knob == 1 : flops >= (D == 64 ? 5.6e9 : 7e9) * (kv_dtype == KVC_F16 ? 0.6 : 1.0);
    }
    std::vector<Tile> tiles;
    tiles.reserve(N);
    long long row = 0, tab = 0;
    wide = 0;
    for (int s = 0; s < N; ++s) {
        const int nq = q_lens[s], nk = kv_lens[s];
        if (tab_off) tab = tab_off[s];
        const long long rows = (long long)nq * group;
        const bool tile = tiled && rows > kTileRows;
        const int cap = !tile ? 16 : rows <= 128 ? 128 : 256;
        const int hstep = std::min(group, cap), tstep = std::max(1, cap / group);
        const int key0 = first_key(nk - nq);  // the first key that any of the new tokens sees
        for (int i = 0; i < nq; i += tstep)
            for (int h = 0; h < group; h += hstep) {
                Tile t{tile ? kKindTile : kKindRows, (int)row + i, std::min(tstep, nq - i), nk - nq + i, h,
                       std::min(hstep, group - h), 0, 0, (int)tab, (int)std::min<long long>(wide, INT_MAX), key0};
                t.j1 = t.pos0 + t.ntok;
                t.j0 = first_key(t.pos0);
                tiles.push_back(t);
            }
        if (tile && kv_dtype != KVC_F16) wide += nk - key0;
        row += nq;
        if (!tab_off) tab += ((long long)nk + BLOCK - 1) / BLOCK;
    }
    records = 0;
    const long long chunk[2] = {stream_chunk(tiles, Hkv, D), tile_chunk(tiles, Hkv, D)};
    units.reserve(tiles.size() + tiles.size() / 4);
    for (const Tile& t : tiles) {
        const int len = t.j1 - t.j0;
        int nc = chunks_of(len, chunk[t.kind == kKindTile]);
        const int step = ((len + nc - 1) / nc + 63) / 64 * 64;
        nc = (len + step - 1) / step;
        const int rows = t.ntok * t.hn;
        for (int c = 0; c < nc; ++c) {
            PlanUnit u{};
            u.f[kFKind] = t.kind;
            u.f[kFRow] = t.row0;
            u.f[kFTok] = t.ntok;
            u.f[kFPos] = t.pos0;
            u.f[kFHead] = t.h0;
            u.f[kFHeads] = t.hn;
            u.f[kFJ0] = t.j0 + c * step;
            u.f[kFJ1] = std::min(t.j1, t.j0 + (c + 1) * step);
            u.f[kFChunk] = c;
            u.f[kFChunks] = nc;
            u.f[kFRec] = nc > 1 ? (int)std::min<long long>(records, INT_MAX) : 0;
            u.f[kFTab] = t.tab;
            u.f[kFWide] = t.wide;
            u.f[kFWideKey] = t.wkey;
            u.cost = (long long)(u.f[kFJ1] - u.f[kFJ0]) * rows;
            units.push_back(u);
        }
        if (nc > 1) records += (long long)nc * rows;
    }
    // a sequence's widened keys in equal shares over its tile units (which follow each other here)
    if (kv_dtype != KVC_F16)
        for (size_t a = 0; a < units.size();) {
            size_t b = a;
            while (b < units.size() && units[b].f[kFKind] == kKindTile && units[b].f[kFTab] == units[a].f[kFTab] &&
                   units[b].f[kFWide] == units[a].f[kFWide])
                ++b;
            const long long first = units[a].f[kFWideKey], n = b > a ? units[b - 1].f[kFJ1] - first : 0;
            for (size_t i = a; i < b; ++i) {
                units[i].f[kFWide0] = (int)(first + n * (long long)(i - a) / (long long)(b - a));
                units[i].f[kFWide1] = (int)(first + n * (long long)(i - a + 1) / (long long)(b - a));
            }
            a = std::max(b, a + 1);
        }
}

// The list's order: tiles first, then by what a unit computes, the longest first (so that the last
// workgroups to start are short).
std::vector<int> unit_order(const std::vector<PlanUnit>& units) {
    std::vector<std::pair<long long, int>> key(units.size());
    for (size_t i = 0; i < units.size(); ++i)
        key[i] = {-(units[i].cost + (units[i].f[kFKind] == kKindTile ? 1LL << 61 : 0)), (int)i};
    std::sort(key.begin(), key.end());
    std::vector<int> order(units.size());
    for (size_t i = 0; i < units.size(); ++i) order[i] = key[i].second;
    return order;
}

template <typename F>
int guard_chunk(F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return set_error(KVC_ERR_NOMEM, "out of host memory");
    } catch (...) {
        return set_error(KVC_ERR_STATE, "unexpected exception");
    }
}

template <int D, int CT>
int launch_chunks_d(const ChunkParams& p, int n_tiles, hipStream_t st) {
    const unsigned Hkv = (unsigned)p.Hkv;
    const unsigned units = (unsigned)(p.n_units - 1), tiles = std::min((unsigned)n_tiles, units);
    bool matrix = false;
    if constexpr (D == 64 || D == 128) {
        matrix = matrix_path(D, p.block);
        if (matrix && tiles > 0) {  // the list's tiles come first
            constexpr bool kWide = CT != kCacheF16;
            if constexpr (kWide) {
                hipLaunchKernelGGL((widen_kernel<D, CT>), dim3(tiles * Hkv, kWidenBlocks), dim3(256), 0, st, p);
                const int rc = hip_check(hipGetLastError(), "chunk attention widening launch");
                if (rc) return rc;
            }
            const dim3 grid(tiles * Hkv), block(kTileWaves * kWave);
            if (p.cap_log2 > 0.f) hipLaunchKernelGGL((chunk_tile_kernel<D, kWide, true>), grid, block, 0, st, p);
            else hipLaunchKernelGGL((chunk_tile_kernel<D, kWide, false>), grid, block, 0, st, p);
            const int rc = hip_check(hipGetLastError(), "chunk attention tile launch");
            if (rc) return rc;
        }
        if (matrix && units > tiles)
            hipLaunchKernelGGL((chunk_stream_kernel<D, CT>), dim3((units - tiles) * Hkv), dim3(kStreamWaves * kWave), 0, st, p);
    }
    if (!matrix) hipLaunchKernelGGL((chunk_rows_kernel<D, CT>), dim3(units * Hkv), dim3(256), 0, st, p);
    int rc = hip_check(hipGetLastError(), "chunk attention launch");
    if (rc || p.n_records == 0) return rc;
    const unsigned split = matrix ? tiles : units;  // (units of 16 rows combine their own)
    if (split == 0) return KVC_OK;
    // a workgroup's share of the rows in about one pass
    const long long passes = ((long long)p.n_records * (D / 4) + 256LL * split - 1) / (256LL * split);
    const dim3 grid(split * Hkv, (unsigned)std::min(8LL, std::max(1LL, passes)));
    if (matrix) hipLaunchKernelGGL((merge_chunks_kernel<D, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((merge_chunks_kernel<D, false>), grid, dim3(256), 0, st, p);
    return hip_check(hipGetLastError(), "chunk attention merge launch");
}

template <int D>
int launch_chunks(const ChunkParams& p, int n_tiles, int kv_dtype, hipStream_t st) {
    if (kv_dtype == KVC_F16) return launch_chunks_d<D, kCacheF16>(p, n_tiles, st);
    if (kv_dtype == KVC_I8) return launch_chunks_d<D, kCacheI8>(p, n_tiles, st);
    return launch_chunks_d<D, kCacheE4M3>(p, n_tiles, st);
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" {

int kvc_chunk_plan(const int* host_q_lens, const int* host_kv_lens, const int* host_tab_off, int N, int Hq, int Hkv,
                   int D, int BLOCK, int kv_dtype, int window, int* work, int capacity, int* n_units, int* n_tiles,
                   int* n_records, int* n_wide) {
    return guard_chunk([&]() -> int {
        int rc = check_shape(Hq, Hkv, D, BLOCK, kv_dtype, window);
        if (rc) return rc;
        if (N < 0 || !n_units || !n_tiles || !n_records || !n_wide) return set_error(KVC_ERR_ARG, "N must be >= 0 and the counts not null");
        if (N > 0 && (!host_q_lens || !host_kv_lens)) return set_error(KVC_ERR_ARG, "null lengths");
        long long rows = 0, blocks = 0;
        for (int s = 0; s < N; ++s) {
            if (host_q_lens[s] < 0 || host_kv_lens[s] < host_q_lens[s])
                return set_error(KVC_ERR_ARG, "sequence " + std::to_string(s) + ": 0 <= q_lens <= kv_lens is needed");
            if (host_tab_off && host_tab_off[s] < 0) return set_error(KVC_ERR_ARG, "negative table offset");
            if (host_tab_off && host_tab_off[s] + ((long long)host_kv_lens[s] + BLOCK - 1) / BLOCK > INT_MAX)
                return set_error(KVC_ERR_UNSUPPORTED, "at most 2^31 - 1 rows and table entries");
            rows += host_q_lens[s];
            blocks += ((long long)host_kv_lens[s] + BLOCK - 1) / BLOCK;
        }
        if (rows > INT_MAX || blocks > INT_MAX) return set_error(KVC_ERR_UNSUPPORTED, "at most 2^31 - 1 rows and table entries");
        std::vector<PlanUnit> units;
        long long records = 0, wide = 0;
        plan_units(host_q_lens, host_kv_lens, host_tab_off, N, Hq, Hkv, D, BLOCK, kv_dtype, window, units, records, wide);
        if (records > INT_MAX || wide > INT_MAX || ((long long)units.size() + 1) * Hkv > INT_MAX)
            return set_error(KVC_ERR_UNSUPPORTED, "the batch needs more than 2^31 - 1 units or partial rows");
        *n_units = (int)units.size() + 1;
        *n_tiles = (int)std::count_if(units.begin(), units.end(), [](const PlanUnit& u) { return u.f[kFKind] == kKindTile; });
        *n_records = (int)records;
        *n_wide = (int)wide;
        if (!work) return KVC_OK;
        if (capacity < *n_units)
            return set_error(KVC_ERR_ARG, "work list too small: " + std::to_string(*n_units) + " entries of 16 ints are needed");
        std::fill(work, work + kChunkInts, 0);
        work[kHdrUnits] = *n_units;
        work[kHdrTiles] = *n_tiles;
        work[kHdrRecords] = *n_records;
        for (const int i : unit_order(units)) {
            work += kChunkInts;
            std::copy(units[i].f, units[i].f + kChunkInts, work);
        }
        return KVC_OK;
    });
}

size_t kvc_chunk_workspace_size(int Hq, int Hkv, int D, int n_records, int n_wide) {
    if (Hq <= 0 || Hkv <= 0 || D <= 0) return 0;
    n_records = std::max(n_records, 0);
    n_wide = std::max(n_wide, 0);
    return acc_bytes(Hkv, D, n_records) + ml_bytes(Hkv, n_records) + ctr_bytes(Hkv, n_records) + 2 * wide_bytes(Hkv, D, n_wide) + factor_bytes(Hkv, n_wide);
}

int kvc_paged_chunk_attn(const void* q, void* out, const void* k_pool, const void* v_pool, const float* kv_scales,
                         const int* table_all, int table_len, const int* work, int n_units, int n_tiles, int n_records,
                         int n_wide, int rows, int Hq, int Hkv, int D, int BLOCK, float scale, float softcap, int window,
                         int kv_dtype, void* workspace, size_t workspace_bytes, kvc_stream_t stream) {
    return guard_chunk([&]() -> int {
        int rc = check_shape(Hq, Hkv, D, BLOCK, kv_dtype, window);
        if (rc) return rc;
        if (rows < 0 || n_units < 0 || n_tiles < 0 || n_records < 0 || n_wide < 0)
            return set_error(KVC_ERR_ARG, "rows and the plan's counts must be >= 0");
        if (!std::isfinite(scale)) return set_error(KVC_ERR_ARG, "scale must be finite");
        if (!(softcap >= 0.f) || !std::isfinite(softcap)) return set_error(KVC_ERR_ARG, "softcap must be >= 0 and finite");
        // (cap - 2 cap / (1 + e^(2x / cap)) is off by cap 2^-23: at 512 a probability by 2^-14)
        if (softcap > 512.f) return set_error(KVC_ERR_UNSUPPORTED, "softcap must be at most 512 (0: none)");
        if (rows == 0 || n_units <= 1) return KVC_OK;
        if ((long long)n_units * Hkv > INT_MAX) return set_error(KVC_ERR_UNSUPPORTED, "at most 2^31 - 1 workgroups");
        if (!q || !out || !k_pool || !v_pool || !table_all || table_len <= 0 || !work)
            return set_error(KVC_ERR_ARG, "null q, out, pool, table or work list");
        auto al = [](const void* x) { return ((uintptr_t)x & 15u) == 0; };
        if (!al(q) || !al(out) || !al(k_pool) || !al(v_pool) || ((uintptr_t)work & 3u))
            return set_error(KVC_ERR_ARG, "q, out and the pools must be 16-byte aligned");
        if (kv_dtype != KVC_F16 && (!kv_scales || ((uintptr_t)kv_scales & 7u)))
            return set_error(KVC_ERR_ARG, "an 8-bit cache needs its scales, 8-byte aligned");
        ChunkParams p{};
        const float log2e = 1.4426950408889634f;
        p.work = work; p.n_units = n_units; p.n_records = n_records; p.n_wide = n_wide;
        p.rows = rows; p.Hq = Hq; p.Hkv = Hkv; p.group = Hq / Hkv; p.block = BLOCK;
        p.table_len = table_len; p.window = window;
        p.scale_log2 = scale * log2e;
        p.cap_log2 = softcap * log2e;
        p.cap_in = softcap > 0.f ? 2.f * scale * log2e / softcap : 0.f;
        if (!std::isfinite(p.scale_log2) || !std::isfinite(p.cap_log2) || !std::isfinite(p.cap_in))
            return set_error(KVC_ERR_ARG, "scale, softcap and scale / softcap must be within fp32's range in log2 units");
        p.q = static_cast<const _Float16*>(q);
        p.out = static_cast<_Float16*>(out);
        p.k = k_pool; p.v = v_pool; p.scales = kv_scales; p.table = table_all;
        if (n_tiles > 0 && kv_dtype != KVC_F16 && n_wide == 0)
            return set_error(KVC_ERR_ARG, "tiles over an 8-bit cache need the plan's n_wide");
        if (n_records > 0 || n_wide > 0) {
            const size_t need = kvc_chunk_workspace_size(Hq, Hkv, D, n_records, n_wide);
            if (!workspace) {
                rc = library_workspace(need, (hipStream_t)stream, &workspace);
                if (rc) return rc;
            } else if (workspace_bytes < need) {
                return set_error(KVC_ERR_WORKSPACE, "workspace too small: need " + std::to_string(need) + " bytes, got " +
                                                        std::to_string(workspace_bytes));
            } else if (!al(workspace)) {
                return set_error(KVC_ERR_ARG, "workspace must be 16-byte aligned");
            }
            char* ws = static_cast<char*>(workspace);
            p.part_acc = reinterpret_cast<float*>(ws);
            ws += acc_bytes(Hkv, D, n_records);
            p.part_ml = reinterpret_cast<float*>(ws);
            ws += ml_bytes(Hkv, n_records);
            p.counters = reinterpret_cast<unsigned long long*>(ws);
            p.epoch = next_epoch();
            ws += ctr_bytes(Hkv, n_records);
            p.wide_k = reinterpret_cast<_Float16*>(ws);
            ws += wide_bytes(Hkv, D, n_wide);
            p.wide_v = reinterpret_cast<_Float16*>(ws);
            p.wide_f = reinterpret_cast<float*>(ws + wide_bytes(Hkv, D, n_wide));
        }
        const hipStream_t st = (hipStream_t)stream;
        switch (D) {
            case 32: return launch_chunks<32>(p, n_tiles, kv_dtype, st);
            case 64: return launch_chunks<64>(p, n_tiles, kv_dtype, st);
            case 128: return launch_chunks<128>(p, n_tiles, kv_dtype, st);
            default: return launch_chunks<256>(p, n_tiles, kv_dtype, st);
        }
    });
}

}  // extern "C"
