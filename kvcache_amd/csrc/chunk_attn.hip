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

// The batch as units.  A sequence whose new tokens make more than kStreamRows rows of a KV head
// is cut into tiles of many rows, others into units of 16.
constexpr int kStreamRows = 32;
constexpr int kChunkKeys = 1024;
void plan_units(const int* q_lens, const int* kv_lens, const int* tab_off, int N, int Hq, int Hkv, int D, int BLOCK,
                int kv_dtype, int window, std::vector<PlanUnit>& units, long long& records, long long& wide) {
    const int group = Hq / Hkv;
    const bool matrix = matrix_path(D, BLOCK);
    std::vector<Tile> tiles;
    long long row = 0, tab = 0;
    wide = 0;
    for (int s = 0; s < N; ++s) {
        const int nq = q_lens[s], nk = kv_lens[s];
        if (tab_off) tab = tab_off[s];
        // the first key that any of the new tokens sees
        const int key0 = window > 0 ? std::max(0, nk - nq - window + 1) / 64 * 64 : 0;
        const bool many = matrix && (long long)nq * group > kStreamRows;
        const int cap = !many ? 16 : (long long)nq * group <= 64 ? 64 : (long long)nq * group <= 1024 ? 128 : 256;
        const int hstep = std::min(group, cap), tstep = std::max(1, cap / group);
        for (int i = 0; i < nq; i += tstep)
            for (int h = 0; h < group; h += hstep) {
                Tile t{many ? kKindTile : kKindRows, (int)row + i, std::min(tstep, nq - i), nk - nq + i, h,
                       std::min(hstep, group - h), 0, 0, (int)tab, (int)std::min<long long>(wide, INT_MAX), key0};
                t.j1 = t.pos0 + t.ntok;
                t.j0 = window > 0 ? std::max(0, t.pos0 - window + 1) / 64 * 64 : 0;
                tiles.push_back(t);
            }
        if (many && kv_dtype != KVC_F16) wide += nk - key0;
        row += nq;
        if (!tab_off) tab += ((long long)nk + BLOCK - 1) / BLOCK;
    }
    records = 0;
    for (const Tile& t : tiles) {
        const int len = t.j1 - t.j0;
        int nc = t.kind == kKindTile ? 1 : std::max(1, (len + kChunkKeys - 1) / kChunkKeys);
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
    std::stable_sort(units.begin(), units.end(), [](const PlanUnit& a, const PlanUnit& b) {
        return a.f[kFKind] != b.f[kFKind] ? a.f[kFKind] > b.f[kFKind] : a.cost > b.cost;
    });
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
            const dim3 grid(tiles * Hkv), block(8 * kWave);
            if (p.cap_log2 > 0.f) hipLaunchKernelGGL((chunk_tile_kernel<D, kWide, true>), grid, block, 0, st, p);
            else hipLaunchKernelGGL((chunk_tile_kernel<D, kWide, false>), grid, block, 0, st, p);
            const int rc = hip_check(hipGetLastError(), "chunk attention tile launch");
            if (rc) return rc;
        }
        if (matrix && units > tiles)
            hipLaunchKernelGGL((chunk_stream_kernel<D, CT>), dim3((units - tiles) * Hkv),
                               dim3(StreamShape<D, CT>::W * kWave), 0, st, p);
    }
    if (!matrix) hipLaunchKernelGGL((chunk_rows_kernel<D, CT>), dim3(units * Hkv), dim3(256), 0, st, p);
    int rc = hip_check(hipGetLastError(), "chunk attention launch");
    if (rc || p.n_records == 0) return rc;
    hipLaunchKernelGGL((merge_chunks_kernel<D>), dim3(units * Hkv), dim3(256), 0, st, p);
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
        for (size_t i = 0; i < units.size(); ++i) std::copy(units[i].f, units[i].f + kChunkInts, work + (i + 1) * kChunkInts);
        return KVC_OK;
    });
}

size_t kvc_chunk_workspace_size(int Hq, int Hkv, int D, int n_records, int n_wide) {
    if (Hq <= 0 || Hkv <= 0 || D <= 0) return 0;
    n_records = std::max(n_records, 0);
    n_wide = std::max(n_wide, 0);
    return acc_bytes(Hkv, D, n_records) + ml_bytes(Hkv, n_records) + 2 * wide_bytes(Hkv, D, n_wide);
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
            p.wide_k = reinterpret_cast<_Float16*>(ws);
            p.wide_v = reinterpret_cast<_Float16*>(ws + wide_bytes(Hkv, D, n_wide));
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
