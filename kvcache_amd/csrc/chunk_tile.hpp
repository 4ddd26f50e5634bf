// chunk_tile.hpp -- chunk attention of many rows on the matrix cores (head_dim 64 / 128).
//
// 8-bit caches: widen_kernel first turns the keys that tiles see into fp16 rows in the workspace.  Every
// tile of a sequence reads all of its keys, so widening them in the tiles costs the more the more
// tiles there are: 2000 tokens of 32 heads behind 6000, D 128, were 316 us with it in the tiles (about
// as many vector instructions as the softmax has).  An error of a score grows with the score, so K is
// exact: the rows hold the code times the leading bits of its scale, as many as fp16 has room for
// behind the code's (4 for int8, 7 for e4m3); the rest of the scale goes in fp32 to the score.  V is
// its code times its scale, rounded once (what an fp16 cache would hold; values beyond fp16's range,
// 65504, become Inf).  Error against 64 bits there 3.0e-4, the output's own rounding 2.1e-4; K rounded
// like V gave 5.0e-4 in 252 instead of 272 us, V exact as well 2.9e-4 in 280 (two multiplications per
// score instead of one).
//
// tile_unit: a workgroup of 8 waves takes 32 QG rows (token, head) of one KV head, QG groups of 32
// rows times KS = 8 / QG key streams.  Keys come in sets of 64, stream ks of a set taking its 64 /
// KS keys.  Wave w brings rows 8 w .. + 7 of a set (one block id, whole rows, rows past the end
// read as zero through the descriptor) into registers while the set before is computed, then into
// LDS: two buffers of K, three of V.  The barrier after which a set may be read stands before the
// last exponentials and P V of the set before it, whose V the next set but one must not overwrite:
// so a wave always has the scores of the next 32 keys to compute under these exponentials.
//
//   S^T[key][row] = K Q^T with v_mfma_f32_32x32x16_f16: a lane holds 16 scores of ONE row
//     (column l % 32), so a row's maximum needs one exchange with lane l ^ 32.
//   softmax: p = 2^(s - reference + kBias), fp32, then fp16.  The reference lags: it moves to the
//     row's maximum when a score passes it by more than 2^kLag (and at a row's first key), so p
//     is at most 2^15, fp16 keeps all its bits down to 2^-21 of the largest, and O is rescaled a
//     few times per row instead of nearly every tile.  The sum is taken over the rounded
//     probabilities (two a v_dot2), the ones O is made of.
//   O^T[dim][row] += V^T P^T: the lane's own probabilities are the operand up to the order of
//     keys, and V^T is read back in that order with the transposing LDS read.
//
// LDS (64 banks, 256 bytes a cycle): K rows as 16-byte chunks permuted so that 16 rows' chunks of one
// dim range lie on different banks, V rows as 32-byte segments permuted so that the two segments of
// four rows that half a wave reads do.
#pragma once
#include "chunk_attn.hpp"

namespace kvc {
namespace {

constexpr float kBias = 7.f, kLag = 8.f;

// Sixteen codes times s as fp16, each rounded once.  int8: the fp16 1024 + (c + 128) comes from a
// byte permutation, and one fma takes 1152 s off again; s has 20 bits at most (leading), so that
// 1152 s is exact.
template <int CT>
__device__ __forceinline__ void scaled_f16(u32x4 c, float s, u32x4 (&out)[2]) {
    const float off = CT == kCacheI8 ? -1152.f * s : 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f16x2 a, b;
        if constexpr (CT == kCacheI8) {
            const unsigned x = c[w] ^ 0x80808080u;
            a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u));
            b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u));
        } else {
            codes_to_f16<CT>(c[w], a, b);
        }
        f16x4 y;
        y[0] = (_Float16)__builtin_fmaf((float)a[0], s, off);
        y[1] = (_Float16)__builtin_fmaf((float)a[1], s, off);
        y[2] = (_Float16)__builtin_fmaf((float)b[0], s, off);
        y[3] = (_Float16)__builtin_fmaf((float)b[1], s, off);
        const u32x2 z = __builtin_bit_cast(u32x2, y);
        out[w >> 1][2 * (w & 1)] = z[0];
        out[w >> 1][2 * (w & 1) + 1] = z[1];
    }
}

// s without all but its leading `bits` bits
__device__ __forceinline__ float leading(float s, int bits) { return __uint_as_float(__float_as_uint(s) & (~0u << (24 - bits))); }

// A tile's share of its sequence's keys, as fp16 rows of the workspace.
constexpr int kWidenBlocks = 16;  // workgroups per tile and KV head
template <int D, int CT>
__global__ __launch_bounds__(256) void widen_kernel(ChunkParams p) {
    constexpr int LPR = D / 16, RPB = 256 / LPR;
    ChunkUnit u;
    if (!chunk_unit(p, u, 0) || u.kind != kKindTile) return;
    const int n = u.w1 - u.w0, per = (n + kWidenBlocks - 1) / kWidenBlocks;
    const int k0 = u.w0 + blockIdx.y * per, k1 = min(k0 + per, u.w1);
    const int l = threadIdx.x % LPR;
    const float kf = p.cap_log2 > 0.f ? p.cap_in : p.scale_log2;
    for (int k = k0 + threadIdx.x / LPR; k < k1; k += RPB) {
        const int b = k / p.block;
        const int id = block_id(p, u, b);
        const size_t row = ((size_t)(unsigned)(id * p.Hkv + u.hk)) * p.block + (k - b * p.block);
        const size_t to = (size_t)u.hk * p.n_wide + u.wide + (k - u.wkey);
        const f32x2 s = *reinterpret_cast<const f32x2*>(p.scales + row * 2);
        const u32x4 ck = *reinterpret_cast<const u32x4*>(static_cast<const char*>(p.k) + row * D + 16 * l);
        const u32x4 cv = *reinterpret_cast<const u32x4*>(static_cast<const char*>(p.v) + row * D + 16 * l);
        u32x4* ko = reinterpret_cast<u32x4*>(p.wide_k + to * D + 16 * l);
        u32x4* vo = reinterpret_cast<u32x4*>(p.wide_v + to * D + 16 * l);
        const float lead = leading(s[0], CT == kCacheI8 ? 4 : 7);
        u32x4 x[2];
        scaled_f16<CT>(ck, lead, x);
        ko[0] = x[0];
        ko[1] = x[1];
        scaled_f16<CT>(cv, leading(s[1], 20), x);
        vo[0] = x[0];
        vo[1] = x[1];
        // (0, subnormal and non-finite scales: all of it is in K)
        if (l == 0) p.wide_f[to] = fabsf(lead) >= FLT_MIN && fabsf(lead) <= FLT_MAX ? s[0] / lead * kf : kf;
    }
}

// S[i] times the f of lane i of the 16 around a lane (one instruction each: a row broadcast is an
// operand's modifier).
template <int I = 0>
__device__ __forceinline__ void scale_scores(f32x16& S, float f) {
    if constexpr (I < 16) {
        S[I] *= __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, f), 0x150 + I, 0xf, 0xf, true));
        scale_scores<I + 1>(S, f);
    }
}

constexpr int kSetKeys = 64;  // keys of an LDS set: 8 rows for each of 8 waves
constexpr int kTileWaves = 8;

template <int D>
struct TileLds {
    char k[2][kSetKeys * D * 2];
    char v[3][kSetKeys * D * 2];
    float kf[3][kSetKeys];  // widened keys: the score's factor
};

// WIDE: keys from the workspace (widen_kernel), else from the pages of an fp16 cache.
template <int D, bool WIDE, int QG, bool CAP>
__device__ __forceinline__ void tile_unit(const ChunkParams& p, const ChunkUnit& u, TileLds<D>& lds) {
    constexpr int W = 8;
    constexpr int SR = kSetKeys / W;         // rows of a set that a wave brings
    constexpr int ROW = D * 2;               // bytes of a row
    constexpr int KS = W / QG;               // key streams
    constexpr int KT = kSetKeys / KS;        // keys per stream and set
    constexpr int NS = KT / 32;              // 32-key subtiles
    constexpr int KD = D / 16;               // MFMA k steps over the head dimension
    constexpr int DT = D / 32;               // 32-dim output tiles
    constexpr int VL = SR * ROW / 1024;      // wave loads per set
    static_assert(NS >= 1 && KS <= 2, "one or two streams of whole subtiles");
    __shared__ float s_ml[QG][32][2];
    __shared__ int s_bad[W];

    const int lane = threadIdx.x & (kWave - 1);
    const int wave = uniform(threadIdx.x >> 6);
    const int qg = wave % QG, ks = wave / QG;
    const int l32 = lane & 31, h = lane >> 5;
    const int j0 = u.j0, j1 = u.j1;
    const int nsets = (j1 - j0 + kSetKeys - 1) / kSetKeys;
    const int bsh = __builtin_ctz((unsigned)p.block), bmask = p.block - 1;
    const char* kb = WIDE ? reinterpret_cast<const char*>(p.wide_k) : static_cast<const char*>(p.k);
    const char* vb = WIDE ? reinterpret_cast<const char*>(p.wide_v) : static_cast<const char*>(p.v);

    // Sets [f0, f1) are seen whole by every row; they come first, then those before them (the
    // window's edge) and after them (the causal one): the i-th set to come is set_at(i).
    const int plast = u.pos0 + u.ntok - 1;
    const int f0 = p.window > 0 ? min(nsets, max(0, plast - p.window + 1 - j0 + kSetKeys - 1) / kSetKeys) : 0;
    const int f1 = max(f0, (min(u.pos0 + 1, j1) - j0) / kSetKeys);
    const int nfull = f1 - f0;
    auto set_at = [&](int i) { return i < nfull ? f0 + i : i - nfull < f0 ? i - nfull : i; };
    // this wave's rows of the i-th set; block ids one set per lane, 64 sets at a time
    auto first_tok = [&](int i) { return j0 + set_at(i) * kSetKeys + SR * wave; };
    int ids = 0;
    auto load_ids = [&](int i) {
        if constexpr (!WIDE) ids = block_id(p, u, min(first_tok(i + lane), j1 - 1) >> bsh);
    };
    auto row_of = [&](int t, int id) -> size_t {
        if constexpr (WIDE) return (size_t)u.hk * p.n_wide + u.wide + (t - u.wkey);
        else return (((size_t)(unsigned)(id * p.Hkv + u.hk)) << bsh) + (t & bmask);
    };
    u32x4 rk[VL], rv[VL];
    float rf = 0.f;  // (of row 8 w + lane, lanes 0 .. 7)
    auto issue = [&](int i) {
        const int t = first_tok(i);
        const int id = WIDE ? 0 : __builtin_amdgcn_readlane(ids, i & (kWave - 1));
        int rows = max(j1 - t, 0);
        asm("" : "+s"(rows));
        const int bytes = min(rows, SR) * ROW;
        const size_t off = row_of(rows > 0 ? t : j0, id) * ROW;
        const __amdgpu_buffer_rsrc_t kr = tile_rsrc(kb + off, bytes), vr = tile_rsrc(vb + off, bytes);
#pragma unroll
        for (int n = 0; n < VL; ++n) rk[n] = buffer_load16(kr, n * 1024 + lane * 16);
#pragma unroll
        for (int n = 0; n < VL; ++n) rv[n] = buffer_load16(vr, n * 1024 + lane * 16);
        if constexpr (WIDE) {
            const __amdgpu_buffer_rsrc_t fr = tile_rsrc(p.wide_f + off / ROW, min(rows, SR) * 4);
            rf = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(fr, lane * 4, 0, 0));
        }
    };
    auto kchunk = [](int r, int ch) { return ch ^ (D == 64 ? (r >> 1) & 7 : r & 15); };
    auto vseg = [](int r, int seg) { return seg ^ (D == 64 ? r & 2 : 2 * (r & 3)); };
    bool bad = false;  // this wave cleared elements of V in sets that some row does not see whole
    auto store = [&](int kb2, int vb3, bool edge) {
        char* kd = lds.k[kb2];
        char* vd = lds.v[vb3];
        if (WIDE && lane < SR) lds.kf[vb3][SR * wave + lane] = rf;
        if (edge && any_nonfinite(rv)) {
            clear_nonfinite(rv);
            bad = true;
        }
#pragma unroll
        for (int n = 0; n < VL; ++n) {
            const int off = n * 1024 + lane * 16;
            const int r = SR * wave + off / ROW, cb = off % ROW;
            *reinterpret_cast<u32x4*>(kd + r * ROW + kchunk(r, cb >> 4) * 16) = rk[n];
            *reinterpret_cast<u32x4*>(vd + r * ROW + vseg(r, cb >> 5) * 32 + (cb & 31)) = rv[n];
        }
    };

    load_ids(0);
    issue(0);
    // q as the B operand: lane l holds row 32 qg + l % 32, dims 16 d + 8 (l / 32) .. + 7
    const int row = 32 * qg + l32, rowc = min(row, u.rows - 1);
    const int pos = u.pos0 + rowc / u.hn;
    f16x8v qb[KD];
    {
        const _Float16* q = p.q + chunk_row(p, u, rowc, D) + 8 * h;
#pragma unroll
        for (int d = 0; d < KD; ++d) qb[d] = *reinterpret_cast<const f16x8v*>(q + 16 * d);
    }
    // paged keys: the score's factor to log2 units, > 0 here (a negative one negates q, exactly; 0: q
    // becomes 0, so that the -Inf of unseen keys stays one)
    const float sl2 = WIDE || CAP || p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
    if (!WIDE && !CAP && p.scale_log2 <= 0.f) {
        const _Float16 f = p.scale_log2 < 0.f ? -1.f : 0.f;
#pragma unroll
        for (int d = 0; d < KD; ++d) qb[d] *= f;
    }

    float ref = 0.f, l = 0.f;    // p = 2^(score - ref); sum of the lane's own keys
    float thr = -FLT_MAX;        // a score above it moves the reference (none met yet: any)
    f32x16 O[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) O[dt][i] = 0.f;

    int ka[KD], va[DT];  // operand addresses within a set
#pragma unroll
    for (int d = 0; d < KD; ++d) ka[d] = (ks * KT + l32) * ROW + kchunk(l32, 2 * d + h) * 16;
    const int vr = 4 * h + ((lane & 15) >> 2);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
        va[dt] = (ks * KT + vr) * ROW + vseg(vr, 2 * dt + ((lane >> 4) & 1)) * 32 + 8 * (lane & 3);

    auto scores = [&](const char* kd, int n) {
        f32x16 S;
#pragma unroll
        for (int i = 0; i < 16; ++i) S[i] = 0.f;
#pragma unroll
        for (int d = 0; d < KD; ++d) {
            const f16x8v a = *reinterpret_cast<const f16x8v*>(kd + ka[d] + 32 * n * ROW);
            S = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qb[d], S, 0, 0, 0);
        }
        return S;
    };
    const int fl = 8 * ((lane & 15) >> 2) + 4 * h + (lane & 3);  // the key whose factor a lane fetches
    // scores in log2 units, those of unseen keys -Inf; the reference moves where one is too far above
    // it.  S[i] is key t0 + 8 (i / 4) + 4 h + i % 4; the subtile's factors begin at kf.
    auto settle = [&](f32x16& S, const float* kf, int t0, auto masked_tag) {
        if constexpr (WIDE) scale_scores(S, kf[fl]);
        // (capped: S becomes w = 1 / (1 + e^(2x / cap)), the score is cap - 2 cap w)
        if constexpr (CAP) {
            const float f = WIDE ? 1.f : p.cap_in;
#pragma unroll
            for (int i = 0; i < 16; ++i) S[i] = __builtin_amdgcn_rcpf(1.f + fast_exp2(S[i] * f));
        }
        constexpr float kNone = CAP ? __builtin_inff() : -__builtin_inff();
        if constexpr (decltype(masked_tag)::value) {
            // seen when low < 8 (i / 4) + i % 4 <= lim
            const int lim = min(pos, j1 - 1) - t0 - 4 * h;
            const int low = (p.window > 0 ? pos - p.window : -1) - t0 - 4 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int c = 8 * (i >> 2) + (i & 3);
                S[i] = c <= lim && c > low ? S[i] : kNone;
            }
        }
        float mx = CAP ? FLT_MAX : -FLT_MAX;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = CAP ? fminf(mx, S[i]) : fmaxf(mx, S[i]);
        if constexpr (CAP) mx = __builtin_fmaf(mx, -2.f * p.cap_log2, p.cap_log2);
        // (rare: said so, since the compiler otherwise copies O for its sake on every tile)
        if (__builtin_expect(__any(mx * sl2 > thr), 0)) {
            mx = max_xor32(mx) * sl2;
            const bool move = mx > thr;
            // (a little further for scores whose last bit is more than 1: p has to stay below 2^16)
            const float to = move ? mx - kBias + fabsf(mx) * 0x1p-22f : ref;
            const float corr = thr > -FLT_MAX ? fast_exp2(ref - to) : 1.f;
            ref = to;
            thr = move ? mx + kLag : thr;
            l *= corr;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) O[dt][i] *= corr;
        }
    };
    // probabilities and P V of a subtile, the n-th of its set
    auto weigh = [&](const f32x16& S, const char* vd, int n) {
        f16x8v pb[2];
        const float off = CAP ? p.cap_log2 - ref : -ref;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int j = 0; j < 8; ++j) pb[t][j] = (_Float16)fast_exp2(__builtin_fmaf(S[8 * t + j], CAP ? -2.f * p.cap_log2 : sl2, off));
            const f16x2 one = {(_Float16)1.f, (_Float16)1.f};
            l = __builtin_amdgcn_fdot2(__builtin_shufflevector(pb[t], pb[t], 0, 1), one, l, false);
            l = __builtin_amdgcn_fdot2(__builtin_shufflevector(pb[t], pb[t], 2, 3), one, l, false);
            l = __builtin_amdgcn_fdot2(__builtin_shufflevector(pb[t], pb[t], 4, 5), one, l, false);
            l = __builtin_amdgcn_fdot2(__builtin_shufflevector(pb[t], pb[t], 6, 7), one, l, false);
        }
        // V^T operand: k slots (h, j) are keys 32 n + 16 t + 8 (j / 4) + 4 h + j % 4, of dim 32 dt
        // + l % 32; two transposing reads of four keys each (16 lanes address four rows of 16
        // dims: lane i row i / 4, dims 4 (i % 4) .. + 3)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const char* vt = vd + va[dt] + (32 * n + 16 * t) * ROW;
                const s16x4v lo = ds_read_tr16(vt), hi = ds_read_tr16(vt + 8 * ROW);
                const f16x8v a = __builtin_bit_cast(f16x8v, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                O[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pb[t], O[dt], 0, 0, 0);
            }
    };

    store(0, 0, nfull == 0);
    issue(1);
    __syncthreads();
    f32x16 S = scores(lds.k[0], 0);
    settle(S, lds.kf[0] + ks * KT, j0 + set_at(0) * kSetKeys + ks * KT, std::true_type{});
    // (the wave that has products to issue goes first: the two waves of a SIMD then take turns with
    // products and settling; 4 x 700 tokens with cap and window 60.6 -> 57.2 us, 2000 behind 6000 1%)
    // One set, whose first scores are there: the next one from its registers into LDS, the one after
    // that into flight; then this one's subtiles, each under the scores of the one after it.
    int v3 = 0;  // the V buffer of the set
    auto set = [&](int i, auto masked_tag) {
        const char* kd = lds.k[i & 1];
        const char* vd = lds.v[v3];
        const float* kf = lds.kf[v3] + ks * KT;
        v3 = v3 == 2 ? 0 : v3 + 1;
        store((i + 1) & 1, v3, decltype(masked_tag)::value);
        if (!WIDE && ((i + 2) & (kWave - 1)) == 0) load_ids(i + 2);
        issue(i + 2);  // (sets past the last read nothing: zero-size descriptors)
        const int t0 = j0 + set_at(i) * kSetKeys + ks * KT;
#pragma unroll
        for (int n = 0; n + 1 < NS; ++n) {
            __builtin_amdgcn_s_setprio(1);
            f32x16 next = scores(kd, n + 1);
            weigh(S, vd, n);
            __builtin_amdgcn_s_setprio(0);
            settle(next, kf + 32 * (n + 1), t0 + 32 * (n + 1), masked_tag);
            S = next;
        }
        __syncthreads();
        __builtin_amdgcn_s_setprio(1);
        f32x16 next = scores(lds.k[(i + 1) & 1], 0);  // (past the last set: rows stored as zero, masked)
        weigh(S, vd, NS - 1);
        __builtin_amdgcn_s_setprio(0);
        settle(next, lds.kf[v3] + ks * KT, j0 + set_at(i + 1) * kSetKeys + ks * KT, masked_tag);
        S = next;
    };
    // sets whose next one is seen whole as well, then the rest (loops of their own: one loop with both
    // forms copied O between them in every set)
    int i = 0;
    for (; i < nfull - 1; ++i) set(i, std::false_type{});
    for (; i < nsets; ++i) set(i, std::true_type{});
    l = sum_xor32(l);
    const float m = thr > -FLT_MAX ? ref : -FLT_MAX;

    auto write = [&](int r, int d0, f32x4 acc, float M, float lt) {
        if (u.nc == 1) {
            const float inv = lt == 0.f ? 0.f : 1.0f / lt;
            f16x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (_Float16)(acc[e] * inv);
            *reinterpret_cast<f16x4*>(p.out + chunk_row(p, u, r, D) + d0) = o;
        } else {
            const size_t rec = (size_t)u.hk * p.n_records + u.rec0 + (size_t)u.c * u.rows + r;
            *reinterpret_cast<f32x4*>(p.part_acc + rec * D + d0) = acc;
            if (d0 == 0) {
                p.part_ml[rec * 2] = M;
                p.part_ml[rec * 2 + 1] = lt;
            }
        }
    };
    // Inf and NaN of V (as staged) of the keys that this lane's row sees, as add_seen_nonfinite
    auto add_bad = [&](f32x4 acc, int d0) {
        if constexpr (!WIDE) return add_seen_nonfinite<D>(p, u, acc, pos, d0);
        for (int j = max(j0, p.window > 0 ? pos - p.window + 1 : 0); j <= min(j1 - 1, pos); ++j) {
            const f16x4 v = *reinterpret_cast<const f16x4*>(p.wide_v + row_of(j, 0) * D + d0);
            const u16x4 bits = __builtin_bit_cast(u16x4, v);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (nonfinite(bits[r])) acc[r] += (float)v[r];
        }
        return acc;
    };
    if (lane == 0) s_bad[wave] = bad;
    __syncthreads();  // (the last set has been read)
    int any_bad = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) any_bad |= s_bad[w];
    // two streams: the second one's (m, l, O) go through LDS to the first one's waves
    static_assert(KS == 1 || QG * 32 * D * 4 <= (int)sizeof(TileLds<D>), "partials fit the buffers");
    f32x4* part = reinterpret_cast<f32x4*>(&lds) + qg * (DT * 4) * kWave + lane;
    float M = m, w0 = 1.f, w1 = 0.f;
    if constexpr (KS == 2) {
        if (ks == 1) {
#pragma unroll
            for (int b = 0; b < DT * 4; ++b)
                part[b * kWave] = f32x4{O[b >> 2][4 * (b & 3)], O[b >> 2][4 * (b & 3) + 1], O[b >> 2][4 * (b & 3) + 2],
                                        O[b >> 2][4 * (b & 3) + 3]};
            if (h == 0) {
                s_ml[qg][l32][0] = m;
                s_ml[qg][l32][1] = l;
            }
        }
        __syncthreads();
        if (ks == 1) return;
        M = fmaxf(m, s_ml[qg][l32][0]);
        w0 = fast_exp2(m - M);
        w1 = fast_exp2(s_ml[qg][l32][0] - M);
        l = l * w0 + s_ml[qg][l32][1] * w1;
    }
    if (row >= u.rows) return;
#pragma unroll
    for (int b = 0; b < DT * 4; ++b) {
        f32x4 acc = {O[b >> 2][4 * (b & 3)], O[b >> 2][4 * (b & 3) + 1], O[b >> 2][4 * (b & 3) + 2], O[b >> 2][4 * (b & 3) + 3]};
        if constexpr (KS == 2) {
            const f32x4 x = part[b * kWave];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = acc[e] * w0 + x[e] * w1;
        }
        const int d0 = 8 * b + 4 * h;
        if (any_bad) acc = add_bad(acc, d0);
        write(row, d0, acc, M, l);
    }
}

template <int D, bool WIDE, bool CAP>
__global__ __launch_bounds__(8 * kWave, D == 64 ? 4 : 2) void chunk_tile_kernel(ChunkParams p) {
    __shared__ __attribute__((aligned(16))) TileLds<D> lds;
    ChunkUnit u;
    if (!chunk_unit(p, u, 0) || u.kind != kKindTile) return;
    if (u.rows <= 128) tile_unit<D, WIDE, 4, CAP>(p, u, lds);
    else if (u.rows <= 256) tile_unit<D, WIDE, 8, CAP>(p, u, lds);
}

}  // namespace
}  // namespace kvc
