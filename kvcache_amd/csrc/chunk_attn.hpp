// chunk_attn.hpp -- attention of a ragged batch of chunks over a paged cache: parameters and
// what its kernels share.
//
// Work list (kvc_chunk_plan): entries of 16 ints, entry 0 the header.  A unit is n_tok
// consecutive tokens of one sequence times hn query heads of each KV head, over keys j0 .. j1-1;
// a workgroup takes one unit of one KV head.  Its rows r = (token i, head g) = (r / hn, r % hn)
// share every K and V row it reads.  A unit whose key range is one of nc > 1 leaves partial rows
// (running maximum in log2 units, sum, unnormalised output): of the units of 16 rows on the matrix
// cores the last one to arrive combines them, of the others merge_chunks_kernel does.
#pragma once
#include "cache8.hpp"

namespace kvc {

constexpr int kChunkInts = 16;
enum ChunkHeader { kHdrUnits = 0, kHdrTiles = 1, kHdrRecords = 2 };
// kFWide..kFWide1 (tiles over an 8-bit cache): the workspace row of key kFWideKey of the sequence,
// and the keys that this unit widens into it
enum ChunkField { kFKind = 0, kFRow = 1, kFTok = 2, kFPos = 3, kFHead = 4, kFHeads = 5, kFJ0 = 6, kFJ1 = 7, kFChunk = 8,
                  kFChunks = 9, kFRec = 10, kFTab = 11, kFWide = 12, kFWideKey = 13, kFWide0 = 14, kFWide1 = 15 };
enum ChunkKind { kKindRows = 0, kKindTile = 1 };

struct ChunkParams {
    const int* work;
    int n_units;            // entries of the list the grid covers, the header included
    int n_records;          // partial rows per KV head that the workspace holds
    int n_wide;             // ... and widened keys
    int rows, Hq, Hkv, group, block;
    int table_len, window;
    unsigned epoch;         // the launch's tag of its arrival counters
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
    unsigned long long* counters;  // [Hkv][n_records]: arrivals of the units whose records begin there
    _Float16* wide_k;       // [Hkv][n_wide][D]
    _Float16* wide_v;
    float* wide_f;          // [Hkv][n_wide]: the score's factor
};

namespace {

struct ChunkUnit {
    int kind, row0, ntok, pos0, h0, hn, j0, j1, c, nc, rec0, tab;
    int wide, wkey, w0, w1;
    int hk;
    int rows;   // ntok * hn
};

// The workgroup's unit, the list's entry 1 + skip + blockIdx.x / Hkv; false past the list's end and
// for entries that do not fit the launch.
__device__ __forceinline__ bool chunk_unit(const ChunkParams& p, ChunkUnit& u, int skip) {
    const int i = (int)(blockIdx.x / (unsigned)p.Hkv) + 1 + skip;
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
    u.wide = e[kFWide];
    u.wkey = e[kFWideKey];
    u.w0 = e[kFWide0];
    u.w1 = e[kFWide1];
    u.hk = (int)(blockIdx.x % (unsigned)p.Hkv);
    u.rows = u.ntok * u.hn;
    return u.row0 >= 0 && u.ntok > 0 && u.row0 <= p.rows - u.ntok && u.h0 >= 0 && u.hn > 0 && u.h0 <= p.group - u.hn &&
           u.j0 >= 0 && u.j0 < u.j1 && u.pos0 >= 0 && u.j1 - u.pos0 <= u.ntok && u.tab >= 0 && u.c >= 0 && u.c < u.nc &&
           (u.nc == 1 || (u.rec0 >= 0 && (long long)u.rec0 + (long long)u.nc * u.rows <= p.n_records)) &&
           (u.kind != kKindTile || p.n_wide == 0 ||
            (u.wide >= 0 && u.wkey >= 0 && u.wkey <= u.j0 && u.w0 >= u.wkey &&
             (long long)u.wide + (max(u.j1, u.w1) - u.wkey) <= p.n_wide));
}

// Block id of the unit's sequence at table position b, bounded by the table (no sum wraps below it).
__device__ __forceinline__ int block_id(const ChunkParams& p, const ChunkUnit& u, int b) {
    const unsigned at = (unsigned)u.tab + (unsigned)b, last = (unsigned)p.table_len - 1u;
    return p.table[at < last ? at : last];
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
    if (!chunk_unit(p, u, 0)) return;
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
            const int id = block_id(p, u, b);
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

// ---------------------------------------------------------------------------------------------
// Few rows (at most 16 R of a KV head: decode steps, short chunks) on the matrix cores.
//
// A wave streams key tiles of its own, W waves of a workgroup taking tiles in turn; the next
// tile's rows are on their way into registers while this one's are computed.
//   S^T[key][row] = K Q^T with v_mfma_f32_16x16x32_f16: the result gives lane l the scores of
//     row l % 16 for keys 4 (l / 16) + r of each 16-key subtile.  8-bit K is read from LDS 16
//     codes at a time and turned into fp16 exactly; lane l's 16 codes are dims 64 j + 16 (l /
//     16) .. + 15, two k steps of the product, and q lies in that order of dims.  The key's
//     scale multiplies the score.
//   softmax online in log2 units, fp32: p = 2^(s - reference).  The reference lags: it moves to the
//     row's maximum when a score passes it by more than kRowLag, so most tiles need no maximum
//     over the row's lanes and no rescaled O (48 sequences of 1 to 300 tokens, 14q/2kv, D 64: 16.1
//     -> 15.7 us).
//   O[row][dim] += P V: P is the lane's own scores' probabilities (keys 4 g + r of two
//     subtiles, g = l / 16), V is read back transposed: 8-bit rows with ds_read_b64_tr_b8 (of
//     16 lanes, lane i receives byte i % 8 of the 8 bytes that lanes 2 j + i / 8 address, j =
//     0 .. 7: one dim of eight keys), fp16 rows with ds_read_b64_tr_b16.  The key's V scale
//     goes onto its probability, in fp32 and before the rounding to fp16, in units of 2^(E - 11)
//     with 2^E above every V scale met so far (O is kept in them): at the reference 2^11, at most
//     2^15, so that fp16 has all its bits down to 2^-25 of the largest (in units of 2^E, V rows of
//     sizes 2^+-9 cost 2^-8 where a row's weight lay on small ones).  fp16 caches: probabilities
//     are kept times 2^11 for the same reason.  8-bit caches: what the rounding to fp16 loses of a
//     probability follows as a second product, so that the output is as exact as its own rounding
//     (2.1e-4 of 64 bits instead of 3.0e-4; 1 to 6% of the time: the mixed batch 15.7 -> 16.6 us).
//     An Inf in an fp16 cache would become NaN by it.
// D 64 takes three waves a SIMD (168 registers): at four it spilled 76 bytes, and 128 single tokens
// of MHA took 20.6 us instead of 17.3, the mixed batch 18.5 instead of 16.1.
// LDS rows are 16-byte pieces permuted by the row, so that the sixteen rows one operand read
// touches at the same piece lie on different banks.
constexpr int kProbBits = 11, kRowLag = 4;  // probabilities (times V scales) at the reference, and how far they pass it

constexpr int kStreamWaves = 4;  // waves of a workgroup

template <int D, int CT>
struct StreamShape {
    static constexpr int CB = kCodeBytes<CT>;
    static constexpr int ROW = D * CB;              // bytes of a cached row
    static constexpr int KT = CB == 1 ? 64 : 32;    // keys per tile
    static constexpr int SUB = KT / 16;             // 16-key subtiles
    static constexpr int VL = 16 * ROW / 1024;      // 1 KiB wave loads per subtile
    static constexpr int KD = D / 32;               // k steps over the head dimension
    static constexpr int NT = D / 16;               // 16-dim output tiles
    static constexpr int kTile = KT * ROW;          // bytes of a K (or V) tile
    static constexpr int W = kStreamWaves;
    // per wave: the K and V tiles, and the keys' factors
    static constexpr int kWaveBytes = 2 * kTile + 2 * KT * 4;
    static constexpr int kBytes = W * kWaveBytes;
};

__device__ __forceinline__ u32x2 ds_read_tr8(const char* p) {
    typedef int v2i __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (__attribute__((address_space(3))) v2i*)(__attribute__((address_space(3))) char*)(const_cast<char*>(p))));
}

// fp16 caches: Inf and NaN in V.  A key that a row does not see has probability 0, and 0 x Inf
// is NaN, so in the tiles that some row does not see whole the elements of V that are not finite
// are staged as 0; a unit that met one adds them to the rows that see their key: acc += the
// elements d0 .. d0 + 3 of V that are Inf or NaN, of the unit's keys that position pos sees.
// (Those of tiles that were seen whole are in acc already and change nothing.)
template <int D>
__device__ __forceinline__ f32x4 add_seen_nonfinite(const ChunkParams& p, const ChunkUnit& u, f32x4 acc, int pos, int d0) {
    const int bsh = __builtin_ctz((unsigned)p.block);
    const int first = max(u.j0, p.window > 0 ? pos - p.window + 1 : 0), last = min(u.j1 - 1, pos);
    for (int j = first; j <= last; ++j) {
        const int id = block_id(p, u, j >> bsh);
        const size_t row = (((size_t)(unsigned)(id * p.Hkv + u.hk)) << bsh) + (j & (p.block - 1));
        const f16x4 v = *reinterpret_cast<const f16x4*>(static_cast<const _Float16*>(p.v) + row * D + d0);
        const u16x4 bits = __builtin_bit_cast(u16x4, v);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (nonfinite(bits[r])) acc[r] += (float)v[r];
    }
    return acc;
}

// Partials that another workgroup of the launch reads: 16 bytes past the caches that are not
// coherent between XCDs, to the device's point of coherence (sc1, what agent-scope accesses use).
constexpr int kCoherent = 16;
__device__ __forceinline__ void store_coherent(__amdgpu_buffer_rsrc_t r, int at, f32x4 x) {
    typedef int v4i __attribute__((ext_vector_type(4)));
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, x), r, at, 0, kCoherent);
}
__device__ __forceinline__ f32x4 load_coherent(__amdgpu_buffer_rsrc_t r, int at) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, kCoherent));
}
__device__ __forceinline__ void store_coherent2(__amdgpu_buffer_rsrc_t r, int at, f32x2 x) {
    typedef int v2i __attribute__((ext_vector_type(2)));
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2i, x), r, at, 0, kCoherent);
}
__device__ __forceinline__ f32x2 load_coherent2(__amdgpu_buffer_rsrc_t r, int at) {
    return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, kCoherent));
}

// Running (M, l, acc) of four dims of a row over chunks c0, c0 + step, .. of its nc, eight in flight;
// at(c): a chunk's record, as (m, l) and the four dims.
struct MergedRow {
    float M = -FLT_MAX, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    template <typename F>
    __device__ __forceinline__ void add(int c0, int step, int nc, F&& at) {
        constexpr int E = 8;
        for (; c0 < nc; c0 += E * step) {
            // (past the count the last chunk's again, with weight 0)
            f32x2 ml[E];
            f32x4 a[E];
#pragma unroll
            for (int e = 0; e < E; ++e) at(min(c0 + e * step, nc - 1), ml[e], a[e]);
            float top = M;
#pragma unroll
            for (int e = 0; e < E; ++e) top = fmaxf(top, ml[e][0]);
            const float w0 = fast_exp2(M - top);
            M = top;
            l *= w0;
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] *= w0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (c0 + e * step >= nc) continue;
                const float w = fast_exp2(ml[e][0] - M);
                l = __builtin_fmaf(w, ml[e][1], l);
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] = __builtin_fmaf(w, a[e][k], acc[k]);
            }
        }
    }
    __device__ __forceinline__ f16x4 out() const {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        f16x4 o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = (_Float16)(acc[k] * inv);
        return o;
    }
};

template <int D, int CT, int R>
__device__ __forceinline__ void stream_unit(const ChunkParams& p, const ChunkUnit& u, char* lds) {
    using Sh = StreamShape<D, CT>;
    constexpr int ROW = Sh::ROW, KT = Sh::KT, SUB = Sh::SUB, VL = Sh::VL, KD = Sh::KD, NT = Sh::NT, W = Sh::W;
    constexpr bool Q8 = CT != kCacheF16;
    const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x >> 6);
    const int n16 = lane & 15, g4 = lane >> 4;
    const int j0 = u.j0, j1 = u.j1;
    const int ntiles = (j1 - j0 + KT - 1) / KT;
    const int kmax = wave < ntiles ? (ntiles - wave + W - 1) / W : 0;
    const int bsh = __builtin_ctz((unsigned)p.block), bmask = p.block - 1;
    const char* kb = static_cast<const char*>(p.k);
    const char* vb = static_cast<const char*>(p.v);

    // block ids of this wave's subtiles, one per lane, 64 at a time
    auto first_tok = [&](int s) { return j0 + (wave + W * (s / SUB)) * KT + 16 * (s % SUB); };
    int ids = 0;
    auto load_ids = [&](int s) {
        const int t = min(first_tok(s + lane), j1 - 1);
        ids = block_id(p, u, t >> bsh);
    };
    struct Tile {
        u32x4 k[SUB][VL], v[SUB][VL];
        f32x2 sc;
    };
    auto issue = [&](int k, Tile& T) {
        const int t0 = j0 + (wave + W * k) * KT;
        if constexpr (Q8) {  // lane = key; the block of a key past the range is its last one
            const int id = __builtin_amdgcn_ds_bpermute(((SUB * k + g4) & (kWave - 1)) << 2, ids);
            const size_t row = (((size_t)(unsigned)(id * p.Hkv + u.hk)) << bsh) + ((t0 + lane) & bmask);
            T.sc = *reinterpret_cast<const f32x2*>(p.scales + row * 2);
        }
#pragma unroll
        for (int h = 0; h < SUB; ++h) {
            const int t = t0 + 16 * h;
            const int id = __builtin_amdgcn_readlane(ids, (SUB * k + h) & (kWave - 1));
            int rows = max(j1 - t, 0);
            asm("" : "+s"(rows));
            const int bytes = min(rows, 16) * ROW;
            const size_t off = ((((size_t)(unsigned)(id * p.Hkv + u.hk)) << bsh) + (t & bmask)) * ROW;
            const __amdgpu_buffer_rsrc_t kr = tile_rsrc(kb + off, bytes), vr = tile_rsrc(vb + off, bytes);
#pragma unroll
            for (int i = 0; i < VL; ++i) T.k[h][i] = buffer_load16(kr, i * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < VL; ++i) T.v[h][i] = buffer_load16(vr, i * 1024 + lane * 16);
        }
    };

    char* kt = lds + wave * Sh::kWaveBytes;
    char* vt = kt + Sh::kTile;
    float* s_k = reinterpret_cast<float*>(vt + Sh::kTile);  // factor of a key's score
    float* s_v = s_k + KT;                                   // and of its probability
    // 16-byte piece of a K row in LDS, and of an 8-bit V row (fp16: 32-byte segment): sixteen rows
    // of one subtile, and the sixteen (eight) rows that half a wave's transposing read touches, lie
    // on different banks (64 banks, 256 bytes a cycle)
    auto piece = [](int r, int c) { return c ^ (ROW == 64 ? (r >> 2) & 3 : ROW == 128 ? (r >> 1) & 7 : r & 15); };
    auto vseg = [](int r, int seg) {
        if constexpr (Q8) return seg ^ (D == 64 ? (r >> 2 & 1) | (r >> 3 & 2) : (r >> 1 & 3) | (r >> 2 & 4));
        else return seg ^ (D == 64 ? (r >> 1) & 3 : r & 7);
    };

    Tile T;
    if (kmax > 0) {
        load_ids(0);
        issue(0, T);
    }
    // q as the B operand: lane l holds row l % 16; 8-bit: dims 64 j + 16 g + 8 e .. + 7 in step 2 j + e
    f16x8v qb[R][KD];
    int pos[R];
#pragma unroll
    for (int a = 0; a < R; ++a) {
        const int r = min(16 * a + n16, u.rows - 1);
        pos[a] = u.pos0 + r / u.hn;
        const _Float16* q = p.q + chunk_row(p, u, r, D);
#pragma unroll
        for (int d = 0; d < KD; ++d)
            qb[a][d] = *reinterpret_cast<const f16x8v*>(q + (Q8 ? 64 * (d >> 1) + 16 * g4 + 8 * (d & 1) : 32 * d + 8 * g4));
    }
    // q has to be there before the loop: counted as under way in it, its loads made every tile wait for
    // the next one's rows before its first product (4 sequences of 8000 to 32768, 14q/2kv: 16.4 us,
    // 15.2 so; at D 128, where HBM is the bound, 200 sequences 73.4 and 74.3)
    if constexpr (D == 64) {
#pragma unroll
        for (int a = 0; a < R; ++a)
#pragma unroll
            for (int d = 0; d < KD; ++d) asm volatile("" : "+v"(qb[a][d]));
    }
    const bool cap = p.cap_log2 > 0.f;
    const float to_log2 = cap ? p.cap_in : p.scale_log2;
    float ref[R], lim[R], l[R];  // lim: a score further above ref moves it (none met yet: any)
    f32x4 O[R][NT];
    int E = -126;                  // V scales met so far are below 2^E
#pragma unroll
    for (int a = 0; a < R; ++a) {
        ref[a] = 0.f;
        lim[a] = -FLT_MAX;
        l[a] = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) O[a][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    bool bad = false;  // this wave cleared elements of V in tiles that some row does not see whole
    // FULL: every key of the tile is seen by every row
    auto consume = [&](int k, auto full_tag) {
        constexpr bool FULL = decltype(full_tag)::value;
        const int t0 = j0 + (wave + W * k) * KT;
        if constexpr (!Q8 && !FULL) {
            bool b = false;
#pragma unroll
            for (int h = 0; h < SUB; ++h) b |= any_nonfinite(T.v[h]);
            if (b) {
                bad = true;
#pragma unroll
                for (int h = 0; h < SUB; ++h) clear_nonfinite(T.v[h]);
            }
        }
        int En = E;
        if constexpr (Q8) {
            float ks = T.sc[0], vs = T.sc[1];
            if (!FULL && t0 + lane >= j1) ks = vs = 0.f;
            float top = max_xor32(max_xor16(fmaxf(fabsf(vs), 0.f)));  // (NaN: no part in it)
            top = fmaxf(top, dpp<0xB1>(top));
            top = fmaxf(top, dpp<0x4E>(top));
            top = fmaxf(top, dpp<0x141>(top));
            top = fmaxf(top, dpp<0x140>(top));
            const int e = top > 0.f ? __builtin_amdgcn_frexp_expf(top) : -126;
            En = uniform(max(E, e));
            s_k[lane] = ks * to_log2;
            s_v[lane] = __builtin_amdgcn_ldexpf(vs, kProbBits - En);
        }
#pragma unroll
        for (int h = 0; h < SUB; ++h)
#pragma unroll
            for (int i = 0; i < VL; ++i) {
                const int off = i * 1024 + lane * 16;
                const int r = 16 * h + off / ROW, cb = off % ROW;
                *reinterpret_cast<u32x4*>(kt + r * ROW + piece(r, cb >> 4) * 16) = T.k[h][i];
                if constexpr (Q8) *reinterpret_cast<u32x4*>(vt + r * ROW + vseg(r, cb >> 4) * 16) = T.v[h][i];
                else *reinterpret_cast<u32x4*>(vt + r * ROW + vseg(r, cb >> 5) * 32 + (cb & 31)) = T.v[h][i];
            }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
        // the next tile is on its way while this one is computed (its ids a new set of 64
        // subtiles now and then)
        if (k + 1 < kmax) {
            if (((SUB * (k + 1)) & (kWave - 1)) == 0) load_ids(SUB * (k + 1));
            issue(k + 1, T);
        }
        f32x4 S[R][SUB];
#pragma unroll
        for (int h = 0; h < SUB; ++h) {
            const int r = 16 * h + n16;
            f16x8v ka[KD];
            if constexpr (Q8) {
#pragma unroll
                for (int j = 0; j < KD / 2; ++j) {
                    const u32x4 c = *reinterpret_cast<const u32x4*>(kt + r * ROW + piece(r, g4 + 4 * j) * 16);
                    ka[2 * j] = codes_to_f16x8<CT>(u32x2{c[0], c[1]});
                    ka[2 * j + 1] = codes_to_f16x8<CT>(u32x2{c[2], c[3]});
                }
            } else {
#pragma unroll
                for (int j = 0; j < KD; ++j)
                    ka[j] = *reinterpret_cast<const f16x8v*>(kt + r * ROW + piece(r, g4 + 4 * j) * 16);
            }
#pragma unroll
            for (int a = 0; a < R; ++a) {
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KD; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[j], qb[a][j], acc, 0, 0, 0);
                S[a][h] = acc;
            }
        }
        f16x8v pa[R][SUB / 2], pl[R][SUB / 2];
#pragma unroll
        for (int a = 0; a < R; ++a) {
            // key t0 + 16 h + 4 g + r is seen when low < 16 h + r <= last
            const int last = min(pos[a], j1 - 1) - t0 - 4 * g4;
            const int low = (p.window > 0 ? pos[a] - p.window : -1) - t0 - 4 * g4;
            auto seen = [&](int i) {
                const int c = 16 * (i >> 2) + (i & 3);
                return FULL || (c <= last && c > low);
            };
            // scores above the reference, in log2 units
            auto each = [&](auto&& f) {
#pragma unroll
                for (int h = 0; h < SUB; ++h) {
                    f32x4 kf;
                    if constexpr (Q8) kf = *reinterpret_cast<const f32x4*>(s_k + 16 * h + 4 * g4);
                    else kf[0] = kf[1] = kf[2] = kf[3] = to_log2;
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[a][h][r] = f(S[a][h][r], kf[r]);
                }
            };
            if (cap) each([&](float x, float f) { return capped(x, f, p.cap_log2) - ref[a]; });
            else each([&](float x, float f) { return __builtin_fmaf(x, f, -ref[a]); });
            float mx = -FLT_MAX;
#pragma unroll
            for (int i = 0; i < 4 * SUB; ++i) {
                const float x = seen(i) ? S[a][i >> 2][i & 3] : -__builtin_inff();
                S[a][i >> 2][i & 3] = x;
                mx = fmaxf(mx, x);
            }
            if (__builtin_expect(__any(mx > lim[a]) || En != E, 0)) {
                mx = max_xor32(max_xor16(mx));
                const bool move = mx > lim[a];
                // (a little further for scores whose last bit is more than 1: p has to stay within fp16)
                const float by = move ? mx + fabsf(ref[a] + mx) * 0x1p-22f : 0.f;
                const float corr = lim[a] > -FLT_MAX ? fast_exp2(-by) : 1.f;
                ref[a] += by;
                lim[a] = move ? (float)kRowLag : lim[a];
                l[a] *= corr;
#pragma unroll
                for (int i = 0; i < 4 * SUB; ++i) S[a][i >> 2][i & 3] -= by;
                const float oc = Q8 ? __builtin_amdgcn_ldexpf(corr, E - En) : corr;
                // row 4 g + r of the output belongs to the lane that holds row 4 g + r of the scores
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float cr = __int_as_float(__builtin_amdgcn_ds_bpermute((4 * g4 + r) << 2, __float_as_int(oc)));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) O[a][nt][r] *= cr;
                }
            }
#pragma unroll
            for (int h = 0; h < SUB; ++h) {
                f32x4 vf;
                if constexpr (Q8) vf = *reinterpret_cast<const f32x4*>(s_v + 16 * h + 4 * g4);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = fast_exp2(Q8 ? S[a][h][r] : S[a][h][r] + (float)kProbBits);
                    l[a] += e;
                    const float x = !Q8 ? e : seen(4 * h + r) ? e * vf[r] : 0.f;
                    pa[a][h >> 1][4 * (h & 1) + r] = (_Float16)x;
                    if constexpr (Q8) pl[a][h >> 1][4 * (h & 1) + r] = (_Float16)(x - (float)(_Float16)x);
                }
            }
        }
        E = En;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            f16x8v vv[SUB / 2];
#pragma unroll
            for (int s = 0; s < SUB / 2; ++s) {
                if constexpr (Q8) {
                    const int j = n16 >> 1, r = 32 * s + (j < 4 ? 4 * g4 + j : 12 + 4 * g4 + j);
                    vv[s] = codes_to_f16x8<CT>(ds_read_tr8(vt + r * ROW + vseg(r, nt) * 16 + 8 * (n16 & 1)));
                } else {
                    const int r = 32 * s + 4 * g4 + (n16 >> 2), cb = 8 * (n16 & 3);
                    const s16x4v lo = ds_read_tr16(vt + r * ROW + vseg(r, nt) * 32 + cb);
                    const s16x4v hi = ds_read_tr16(vt + (r + 16) * ROW + vseg(r + 16, nt) * 32 + cb);
                    vv[s] = __builtin_bit_cast(f16x8v, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                }
            }
#pragma unroll
            for (int a = 0; a < R; ++a) {
#pragma unroll
                for (int s = 0; s < SUB / 2; ++s) {
                    O[a][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pa[a][s], vv[s], O[a][nt], 0, 0, 0);
                    if constexpr (Q8) O[a][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[a][s], vv[s], O[a][nt], 0, 0, 0);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
    };
    const int plast = u.pos0 + u.ntok - 1;
    // tiles that every row sees whole, between those of the window's edge and of the causal one
    // (loops of their own: one loop with both forms kept the registers of either through both)
    auto tiles_to = [&](int keys) {  // this wave's tiles that begin before j0 + keys
        const int n = max(0, (keys + KT - 1) / KT);
        return min(kmax, n > wave ? (n - wave + W - 1) / W : 0);
    };
    const int whole = min(u.pos0 + 1, j1) - j0;  // keys that every row's position reaches
    const int kf0 = p.window > 0 ? tiles_to(plast - p.window + 1 - j0) : 0;
    const int kf1 = max(kf0, tiles_to(whole / KT * KT));
    int k = 0;
    for (int end = kf0;;) {
        for (; k < end; ++k) consume(k, std::false_type{});
        if (end == kmax) break;
        for (; k < kf1; ++k) consume(k, std::true_type{});
        end = kmax;
    }

    // the waves' (m, l, O) through LDS, each over its own tiles; rows of dims are then summed
    static_assert(16 * R * D * 4 <= 2 * Sh::kTile, "partials fit the tiles");
    const int nwa = min(W, ntiles);
    __shared__ float s_ml[Sh::W][16 * R][3];
    __shared__ int s_bad[Sh::W];
    if (lane == 0) s_bad[wave] = bad;
    if (wave < nwa) {
        float* acc = reinterpret_cast<float*>(kt);
#pragma unroll
        for (int a = 0; a < R; ++a) {
            const float lt = sum_xor32(sum_xor16(l[a]));
            if (lane < 16) {
                s_ml[wave][16 * a + lane][0] = lim[a] > -FLT_MAX ? ref[a] : -FLT_MAX;
                s_ml[wave][16 * a + lane][1] = lt;
                s_ml[wave][16 * a + lane][2] = Q8 ? __builtin_amdgcn_ldexpf(1.f, E - kProbBits) : 1.f;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[(16 * a + 4 * g4 + r) * D + n16 + 16 * nt] = O[a][nt][r];
        }
    }
    __syncthreads();
    int any_bad = 0;
    if constexpr (!Q8) {
#pragma unroll
        for (int w = 0; w < W; ++w) any_bad |= s_bad[w];
    }
    // (nc rows * D floats: below 2^31 bytes in every plan; what a list of other counts reaches is in bounds)
    const size_t first = (size_t)u.hk * p.n_records + u.rec0;
    const int recs = u.nc == 1 ? 0 : min(u.nc, (1 << 20) / u.rows) * u.rows;
    const __amdgpu_buffer_rsrc_t ar = tile_rsrc(p.part_acc + first * D, recs * D * 4), mr = tile_rsrc(p.part_ml + first * 2, recs * 8);
    for (int idx = threadIdx.x; idx < u.rows * (D / 4); idx += W * kWave) {
        const int r = idx / (D / 4), d = idx % (D / 4) * 4;
        float M = -FLT_MAX;
        for (int w = 0; w < nwa; ++w) M = fmaxf(M, s_ml[w][r][0]);
        float lt = 0.f;
        f32x4 at = {0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < nwa; ++w) {
            const float wl = fast_exp2(s_ml[w][r][0] - M), wa = wl * s_ml[w][r][2];
            lt = __builtin_fmaf(wl, s_ml[w][r][1], lt);
            const f32x4 x = *reinterpret_cast<const f32x4*>(lds + w * Sh::kWaveBytes + (r * D + d) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) at[e] = __builtin_fmaf(wa, x[e], at[e]);
        }
        if (any_bad) at = add_seen_nonfinite<D>(p, u, at, u.pos0 + r / u.hn, d);
        if (u.nc == 1) {
            const float inv = lt == 0.f ? 0.f : 1.0f / lt;
            f16x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (_Float16)(at[e] * inv);
            *reinterpret_cast<f16x4*>(p.out + chunk_row(p, u, r, D) + d) = o;
        } else {
            const int rec = u.c * u.rows + r;
            store_coherent(ar, (rec * D + d) * 4, at);
            if (d == 0) store_coherent2(mr, rec * 8, f32x2{M, lt});
        }
    }
    if (u.nc == 1) return;

    // The last of the nc units to arrive combines their partials, always in the order of the chunks.
    // Its threads are 16-byte pieces of the rows times as many groups of chunks as there is room for.
    __shared__ int s_last;
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);  // this wave's partials are written
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    unsigned long long* ctr = p.counters + (size_t)u.hk * p.n_records + u.rec0;
    if (threadIdx.x == 0) s_last = arrive(ctr, p.epoch) == (unsigned)(u.nc - 1);
    __syncthreads();
    if (!s_last) return;
    constexpr int TD = D / 4, NTH = W * kWave;
    const int items = u.rows * TD;
    int groups = 1;
    while (2 * groups * items <= NTH && 4 * groups < u.nc) groups *= 2;
    f32x4* s_acc = reinterpret_cast<f32x4*>(lds);
    f32x2* s_wl = reinterpret_cast<f32x2*>(lds + NTH * sizeof(f32x4));
    static_assert(NTH * 24 <= Sh::kBytes, "the groups' sums fit the tiles");
    for (int i0 = 0; i0 < items; i0 += NTH / groups) {
        const int g = groups == 1 ? 0 : threadIdx.x / items, i = i0 + threadIdx.x - g * items;
        const bool on = g < groups && i < items;
        const int r = i / TD, d = i % TD * 4;
        MergedRow x;
        if (on)
            x.add(g, groups, u.nc, [&](int c, f32x2& ml, f32x4& a) {
                const int rec = c * u.rows + r;
                ml = load_coherent2(mr, rec * 8);
                a = load_coherent(ar, (rec * D + d) * 4);
            });
        if (groups > 1) {  // (then one pass covers every item)
            s_acc[threadIdx.x] = x.acc;
            s_wl[threadIdx.x] = f32x2{x.M, x.l};
            __syncthreads();
            x = MergedRow{};
            if (g == 0)
                x.add(0, 1, groups, [&](int c, f32x2& ml, f32x4& a) {
                    ml = s_wl[c * items + threadIdx.x];
                    a = s_acc[c * items + threadIdx.x];
                });
        }
        if (on && g == 0) *reinterpret_cast<f16x4*>(p.out + chunk_row(p, u, r, D) + d) = x.out();
    }
    if (threadIdx.x == 0) __hip_atomic_store(ctr, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int D, int CT>
__global__ __launch_bounds__(kStreamWaves * kWave, D == 64 ? 3 : 2) void chunk_stream_kernel(ChunkParams p) {
    __shared__ __attribute__((aligned(16))) char lds[StreamShape<D, CT>::kBytes];
    ChunkUnit u;
    if (!chunk_unit(p, u, max(p.work[kHdrTiles], 0)) || u.kind != kKindRows) return;
    if (u.rows <= 16) stream_unit<D, CT, 1>(p, u, lds);
}

// Partial rows of the units with nc > 1 as output rows: out = sum_c 2^(m_c - M) acc_c / sum_c
// 2^(m_c - M) l_c.  A thread takes four dims of a row over all its chunks; the workgroups of a tile's
// nc units (times gridDim.y) share its rows.  TILES: of the tiles only.
template <int D, bool TILES>
__global__ __launch_bounds__(256) void merge_chunks_kernel(ChunkParams p) {
    constexpr int TD = D / 4;
    ChunkUnit u;
    if (!chunk_unit(p, u, 0) || u.nc == 1 || (TILES && u.kind != kKindTile)) return;
    const size_t head = (size_t)u.hk * p.n_records + u.rec0;
    for (int i = (blockIdx.y * u.nc + u.c) * 256 + threadIdx.x; i < u.rows * TD; i += gridDim.y * u.nc * 256) {
        const int r = i / TD, d = i % TD * 4;
        MergedRow x;
        x.add(0, 1, u.nc, [&](int c, f32x2& ml, f32x4& a) {
            const size_t rec = head + (size_t)c * u.rows + r;
            ml = *reinterpret_cast<const f32x2*>(p.part_ml + rec * 2);
            a = *reinterpret_cast<const f32x4*>(p.part_acc + rec * D + d);
        });
        *reinterpret_cast<f16x4*>(p.out + chunk_row(p, u, r, D) + d) = x.out();
    }
}

}  // namespace
}  // namespace kvc
