// chunk_attn.hpp -- attention of a ragged batch of chunks over a paged cache: parameters and
// what its kernels share.
//
// Work list (kvc_chunk_plan): entries of 16 ints, entry 0 the header.  A unit is n_tok
// consecutive tokens of one sequence times hn query heads of each KV head, over keys j0 .. j1-1;
// a workgroup takes one unit of one KV head.  Its rows r = (token i, head g) = (r / hn, r % hn)
// share every K and V row it reads.  A unit whose key range is one of nc > 1 leaves partial rows
// (running maximum in log2 units, sum, unnormalised output) that merge_chunks combines.
#pragma once
#include "cache8.hpp"

namespace kvc {

constexpr int kChunkInts = 16;
enum ChunkHeader { kHdrUnits = 0, kHdrTiles = 1, kHdrRecords = 2 };
enum ChunkField { kFKind = 0, kFRow = 1, kFTok = 2, kFPos = 3, kFHead = 4, kFHeads = 5, kFJ0 = 6, kFJ1 = 7, kFChunk = 8,
                  kFChunks = 9, kFRec = 10, kFTab = 11 };
enum ChunkKind { kKindRows = 0, kKindTile = 1 };

struct ChunkParams {
    const int* work;
    int n_units;            // entries of the list the grid covers, the header included
    int n_records;          // partial rows per KV head that the workspace holds
    int rows, Hq, Hkv, group, block;
    int table_len, window;
    float scale_log2;       // softmax scale * log2(e)
    float cap_log2;         // softcap * log2(e), 0: none
    float cap_in;           // score -> argument of the cap's exponential: 2 * scale * log2(e) / softcap
    const _Float16* q;
    _Float16* out;
    const void* k;
    const void* v;
    const float* scales;    // [num_blocks, Hkv, BLOCK, {k, v}]
    const int* table;
    float* part_acc;        // [Hkv][n_records][D]
    float* part_ml;         // [Hkv][n_records][2]
};

namespace {

struct ChunkUnit {
    int kind, row0, ntok, pos0, h0, hn, j0, j1, c, nc, rec0, tab;
    int hk;
    int rows;   // ntok * hn
};

// The workgroup's unit; false past the list's end and for entries that do not fit the launch.
__device__ __forceinline__ bool chunk_unit(const ChunkParams& p, ChunkUnit& u) {
    const int i = (int)(blockIdx.x / (unsigned)p.Hkv) + 1;
    if (i >= min(p.work[kHdrUnits], p.n_units)) return false;
    const int* e = p.work + (size_t)i * kChunkInts;
    u.kind = e[kFKind];
    u.row0 = e[kFRow];
    u.ntok = e[kFTok];
    u.pos0 = e[kFPos];
    u.h0 = e[kFHead];
    u.hn = e[kFHeads];
    u.j0 = e[kFJ0];
    u.j1 = e[kFJ1];
    u.c = e[kFChunk];
    u.nc = e[kFChunks];
    u.rec0 = e[kFRec];
    u.tab = e[kFTab];
    u.hk = (int)(blockIdx.x % (unsigned)p.Hkv);
    u.rows = u.ntok * u.hn;
    return u.row0 >= 0 && u.ntok > 0 && u.row0 <= p.rows - u.ntok && u.h0 >= 0 && u.hn > 0 && u.h0 <= p.group - u.hn &&
           u.j0 >= 0 && u.pos0 >= 0 && u.tab >= 0 && u.c >= 0 && u.c < u.nc &&
           (u.nc == 1 || (u.rec0 >= 0 && (long long)u.rec0 + (long long)u.nc * u.rows <= p.n_records));
}

// Element offset of row r of the unit in q and out.
__device__ __forceinline__ size_t chunk_row(const ChunkParams& p, const ChunkUnit& u, int r, int D) {
    const int i = r / u.hn;
    return ((size_t)(u.row0 + i) * p.Hq + u.hk * p.group + u.h0 + (r - i * u.hn)) * D;
}

// The capped score in log2 units: cap tanh(x / cap) = cap (1 - 2 / (1 + e^(2x / cap))).
__device__ __forceinline__ float capped(float s, float cap_in, float cap_log2) {
    const float e = fast_exp2(s * cap_in);
    return cap_log2 - 2.f * cap_log2 * __builtin_amdgcn_rcpf(1.f + e);
}

// Any head_dim and block size: a wave takes the unit's rows one at a time, a lane a key.  The
// dot products read K rows lane by lane, in pieces of 16 bytes; then lanes are dims and the keys'
// probabilities are broadcast to them.  Keys outside a row's range are never read.
template <int D, int CT>
__global__ __launch_bounds__(256) void chunk_rows_kernel(ChunkParams p) {
    constexpr int CB = kCodeBytes<CT>;
    constexpr int NJ = (D + kWave - 1) / kWave;
    __shared__ float s_q[4][D];
    ChunkUnit u;
    if (!chunk_unit(p, u)) return;
    const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x >> 6);
    for (int r = wave; r < u.rows; r += 4) {
        const size_t qo = chunk_row(p, u, r, D);
        const int pos = u.pos0 + r / u.hn;
        __builtin_amdgcn_wave_barrier();
        for (int d = lane; d < D; d += kWave) s_q[wave][d] = (float)p.q[qo + d];
        __builtin_amdgcn_wave_barrier();
        const int lo = max(u.j0, p.window > 0 ? pos - p.window + 1 : 0), hi = min(u.j1, pos + 1);
        float m = -FLT_MAX, l = 0.f, acc[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j] = 0.f;
        for (int k0 = lo; k0 < hi; k0 += kWave) {
            const int n = min(kWave, hi - k0);
            const int key = k0 + min(lane, n - 1);
            const int b = key / p.block;
            const int id = p.table[min(u.tab + b, p.table_len - 1)];
            const size_t row = ((size_t)id * p.Hkv + u.hk) * p.block + (key - b * p.block);
            const char* kr = static_cast<const char*>(p.k) + row * (D * CB);
            float s = 0.f;
            for (int d = 0; d < D; d += 8) {
                f16x8 x;
                if constexpr (CT == kCacheF16) x = *reinterpret_cast<const f16x8*>(kr + d * 2);
                else x = codes_to_f16x8<CT>(*reinterpret_cast<const u32x2*>(kr + d));
#pragma unroll
                for (int e = 0; e < 8; ++e) s = __builtin_fmaf((float)x[e], s_q[wave][d + e], s);
            }
            float vs = 1.f;
            if constexpr (CT != kCacheF16) {
                s *= p.scales[row * 2];
                vs = p.scales[row * 2 + 1];
            }
            s = p.cap_log2 > 0.f ? capped(s, p.cap_in, p.cap_log2) : s * p.scale_log2;
            float mx = lane < n ? s : -FLT_MAX;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, shfl_xor(mx, o));
            const float mn = fmaxf(m, mx), corr = fast_exp2(m - mn);
            m = mn;
            const float e = lane < n ? fast_exp2(s - mn) : 0.f;
            l = __builtin_fmaf(l, corr, e);
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[j] *= corr;
            const float pv = e * vs;
            for (int i = 0; i < n; ++i) {
                const float pi = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(pv), i));
                const size_t ri = (size_t)(unsigned)__builtin_amdgcn_readlane((int)row, i) |
                                  (size_t)(unsigned)__builtin_amdgcn_readlane((int)(row >> 32), i) << 32;
                const char* vr = static_cast<const char*>(p.v) + ri * (D * CB);
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int d = min(lane + j * kWave, D - 1);
                    float x;
                    if constexpr (CT == kCacheF16) x = (float)reinterpret_cast<const _Float16*>(vr)[d];
                    else if constexpr (CT == kCacheI8) x = (float)reinterpret_cast<const signed char*>(vr)[d];
                    else x = __builtin_amdgcn_cvt_f32_fp8(reinterpret_cast<const unsigned char*>(vr)[d], 0);
                    acc[j] = __builtin_fmaf(pi, x, acc[j]);
                }
            }
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) l += shfl_xor(l, o);
        if (u.nc == 1) {
            const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                if (lane + j * kWave < D) p.out[qo + lane + j * kWave] = (_Float16)(acc[j] * inv);
        } else {
            const size_t rec = (size_t)u.hk * p.n_records + u.rec0 + (size_t)u.c * u.rows + r;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                if (lane + j * kWave < D) p.part_acc[rec * D + lane + j * kWave] = acc[j];
            if (lane == 0) {
                p.part_ml[rec * 2] = m;
                p.part_ml[rec * 2 + 1] = l;
            }
        }
    }
}

// Partial rows of the units with nc > 1 as output rows: out = sum_c 2^(m_c - M) acc_c / sum_c
// 2^(m_c - M) l_c.  The workgroup of a unit's first chunk takes its rows, a wave one at a time.
template <int D>
__global__ __launch_bounds__(256) void merge_chunks_kernel(ChunkParams p) {
    constexpr int NJ = (D + kWave - 1) / kWave;
    ChunkUnit u;
    if (!chunk_unit(p, u) || u.nc == 1 || u.c != 0) return;
    const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x >> 6);
    for (int r = wave; r < u.rows; r += 4) {
        const size_t rec0 = (size_t)u.hk * p.n_records + u.rec0 + r;
        float M = -FLT_MAX;
        for (int c = 0; c < u.nc; ++c) M = fmaxf(M, p.part_ml[(rec0 + (size_t)c * u.rows) * 2]);
        float l = 0.f, acc[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j] = 0.f;
        for (int c = 0; c < u.nc; ++c) {
            const size_t rec = rec0 + (size_t)c * u.rows;
            const float w = fast_exp2(p.part_ml[rec * 2] - M);
            l = __builtin_fmaf(w, p.part_ml[rec * 2 + 1], l);
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[j] = __builtin_fmaf(w, p.part_acc[rec * D + min(lane + j * kWave, D - 1)], acc[j]);
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        const size_t o = chunk_row(p, u, r, D);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            if (lane + j * kWave < D) p.out[o + lane + j * kWave] = (_Float16)(acc[j] * inv);
    }
}

}  // namespace
}  // namespace kvc
