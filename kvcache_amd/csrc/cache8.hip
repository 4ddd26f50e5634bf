// cache8.hip -- rows of K and V on their way into a paged cache that holds 8-bit codes (or
// fp16), and back: the norm of every query and key head, the rotary position and the cache
// write in one pass; the quantised write alone; the read.
//
// All three move rows: what bounds them is memory, and what is done to a row on the way is
// done in its lanes' registers.  A head row of D values belongs to D / 16 lanes, each holding
// eight values of the row's first half and the eight of its second half that rotate with
// them, so the rotation needs no exchange; the sum of squares (norm) and the largest
// magnitude (scale) take log2(D / 16) register exchanges.
//
// Angles: position times frequency has up to 2^31 turns, more than fp32 resolves from a few
// thousand on (position 1e5: 6e-3 rad).  Turns are counted in fp64 and reduced to a fraction
// of one, from which sine and cosine are taken in fp32, what the fraction loses in fp32 added to
// first order: one (position, frequency) pair per thread and token, shared by all heads through LDS.
//
// A code whose value lies next to a rounding boundary flips with the value's error (e4m3: by 2^-3
// of it), so the roundings on the way are few: see values_to_codes for the quotient.  8192 tokens,
// 32q/8kv, D 128, e4m3: 13 of 8.4 million codes of K are not those of 64 bits, 33 without these.
#include "cache8.hpp"

namespace kvc {
namespace {

constexpr int kRowThreads = 256;

struct RopeWriteParams {
    _Float16* q;
    void* k_pool;
    void* v_pool;
    float* scales;
    const _Float16* qkv;
    long long row_stride;
    const int* pos;
    const int* slots;
    const _Float16* q_norm;
    const _Float16* k_norm;
    float eps;
    double log2_theta;
    int M, Hq, Hkv, block, tokens;  // tokens: per workgroup
};

// The two vectors of a lane into a pool row (16 or 8 bytes each); the row's scale.
template <int D, int CT>
__device__ __forceinline__ float store_row(void* pool, size_t row, int l, const float (&a)[8], const float (&b)[8]) {
    if constexpr (CT == kCacheF16) {
        _Float16* o = static_cast<_Float16*>(pool) + row * D + 8 * l;
        *reinterpret_cast<u32x4*>(o) = Traits<_Float16>::from_float(a);
        *reinterpret_cast<u32x4*>(o + D / 2) = Traits<_Float16>::from_float(b);
        return 1.f;
    } else {
        unsigned mx = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = umax(mx, umax(abs_bits(a[e]), abs_bits(b[e])));
        mx = group_umax<D / 16>(mx);
        float s;
        f32x2 inv;
        row_scale<CT>(mx, s, inv);
        unsigned char* o = static_cast<unsigned char*>(pool) + row * D + 8 * l;
        *reinterpret_cast<u32x2*>(o) = values_to_codes<CT>(a, inv);
        *reinterpret_cast<u32x2*>(o + D / 2) = values_to_codes<CT>(b, inv);
        return s;
    }
}

template <int D, int CT>
__global__ __launch_bounds__(kRowThreads) void norm_rope_write_kernel(RopeWriteParams p) {
    constexpr int LPR = D / 16;                 // lanes per head row
    constexpr int RPB = kRowThreads / LPR;      // head rows per pass of the workgroup
    constexpr int HD = D / 2;
    extern __shared__ f32x2 s_cs[];             // [tokens][HD] (cos, sin)
    const int r0 = blockIdx.x * p.tokens;
    const int nt = min(p.tokens, p.M - r0);
    const int heads = p.Hq + 2 * p.Hkv;
    const int l = threadIdx.x % LPR;
    for (int i = threadIdx.x; i < nt * HD; i += kRowThreads) {
        const int t = i % HD;
        const double f = exp2(-p.log2_theta * (2.0 * t / D)) * 0.15915494309189535;  // turns per position
        const double x = (double)p.pos[r0 + i / HD] * f;
        const double turn = 2.0 * (x - rint(x));
        const float near = (float)turn, rest = 3.14159265f * (float)(turn - (double)near);
        float s, c;
        sincospif(near, &s, &c);
        s_cs[i] = f32x2{__builtin_fmaf(-s, rest, c), __builtin_fmaf(c, rest, s)};
    }
    __syncthreads();
    for (int it = threadIdx.x / LPR; it < nt * heads; it += RPB) {
        const int i = it / heads, h = it - i * heads;
        const int r = r0 + i;
        const _Float16* x = p.qkv + (size_t)r * p.row_stride + (size_t)h * D + 8 * l;
        float a[8], b[8];
        Traits<_Float16>::to_float(*reinterpret_cast<const u32x4*>(x), a);
        Traits<_Float16>::to_float(*reinterpret_cast<const u32x4*>(x + HD), b);
        const int slot = h >= p.Hq ? p.slots[r] : 0;
        if (h < p.Hq + p.Hkv) {
            const _Float16* w = h < p.Hq ? p.q_norm : p.k_norm;
            if (w) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(a[e], a[e], __builtin_fmaf(b[e], b[e], ss));
                ss = group_sum<LPR>(ss);
                const float inv = 1.0f / sqrtf(ss / (float)D + p.eps);
                float wa[8], wb[8];
                Traits<_Float16>::to_float(*reinterpret_cast<const u32x4*>(w + 8 * l), wa);
                Traits<_Float16>::to_float(*reinterpret_cast<const u32x4*>(w + HD + 8 * l), wb);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    a[e] = a[e] * wa[e] * inv;  // (the first product is exact)
                    b[e] = b[e] * wb[e] * inv;
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const f32x2 cs = s_cs[i * HD + 8 * l + e];
                const float u = a[e], v = b[e];
                a[e] = u * cs[0] - v * cs[1];
                b[e] = v * cs[0] + u * cs[1];
            }
        }
        if (h < p.Hq) {
            _Float16* o = p.q + ((size_t)r * p.Hq + h) * D + 8 * l;
            *reinterpret_cast<u32x4*>(o) = Traits<_Float16>::from_float(a);
            *reinterpret_cast<u32x4*>(o + HD) = Traits<_Float16>::from_float(b);
        } else if (slot >= 0) {  // (the same for all lanes of a row)
            const bool is_v = h >= p.Hq + p.Hkv;
            const int hk = h - p.Hq - (is_v ? p.Hkv : 0);
            const int blk = slot / p.block;
            const size_t row = ((size_t)blk * p.Hkv + hk) * p.block + (slot - blk * p.block);
            const float s = store_row<D, CT>(is_v ? p.v_pool : p.k_pool, row, l, a, b);
            if (CT != kCacheF16 && l == 0) p.scales[row * 2 + is_v] = s;
        }
    }
}

struct RowsParams {
    const void* k;   // rows [rows, Hkv, D] (written to where the cache is read)
    const void* v;
    void* k_pool;
    void* v_pool;
    float* scales;
    const int* slots;
    int rows, Hkv, block;
};

// Eight values at element d of row `row`, and back.
template <typename T>
__device__ __forceinline__ void load8(const void* base, size_t at, float (&f)[8]) {
    if constexpr (sizeof(T) == 2) {
        Traits<_Float16>::to_float(*reinterpret_cast<const u32x4*>(static_cast<const _Float16*>(base) + at), f);
    } else {
        const f32x4* x = reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + at);
        const f32x4 u = x[0], v = x[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = u[e], f[4 + e] = v[e];
    }
}
template <typename T>
__device__ __forceinline__ void store8(void* base, size_t at, const float (&f)[8]) {
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<u32x4*>(static_cast<_Float16*>(base) + at) = Traits<_Float16>::from_float(f);
    } else {
        f32x4* x = reinterpret_cast<f32x4*>(static_cast<float*>(base) + at);
        x[0] = f32x4{f[0], f[1], f[2], f[3]};
        x[1] = f32x4{f[4], f[5], f[6], f[7]};
    }
}

// A workgroup: kRowThreads / LPR consecutive tokens of one head, K and V of a token in one thread (the
// rows of a block and its scales then leave as whole lines).  40009 tokens of 8 heads, D 128, int8,
// written and read back, 497 MB: 105 us, of 99 at the rate of a large copy; one row of K or V per
// thread, head after head, 121 us (scales in lines that several XCDs write).
template <int LPR>
__device__ __forceinline__ bool row_of(const RowsParams& p, int& r, int& hk, int& l) {
    const unsigned chunk = blockIdx.x / (unsigned)p.Hkv;
    hk = (int)(blockIdx.x - chunk * (unsigned)p.Hkv);
    r = (int)(chunk * (kRowThreads / LPR) + threadIdx.x / LPR);
    l = threadIdx.x % LPR;
    return r < p.rows;
}
__device__ __forceinline__ size_t pool_row(const RowsParams& p, int slot, int hk) {
    const int blk = slot / p.block;
    return ((size_t)blk * p.Hkv + hk) * p.block + (slot - blk * p.block);
}

template <typename T, int D, int CT>
__global__ __launch_bounds__(kRowThreads) void write_q8_kernel(RowsParams p) {
    int r, hk, l;
    if (!row_of<D / 16>(p, r, hk, l)) return;
    const int slot = p.slots[r];
    const size_t src = ((size_t)r * p.Hkv + hk) * D + 8 * l;
    float k0[8], k1[8], v0[8], v1[8];
    load8<T>(p.k, src, k0);
    load8<T>(p.k, src + D / 2, k1);
    load8<T>(p.v, src, v0);
    load8<T>(p.v, src + D / 2, v1);
    if (slot < 0) return;
    const size_t row = pool_row(p, slot, hk);
    f32x2 s;
    s[0] = store_row<D, CT>(p.k_pool, row, l, k0, k1);
    s[1] = store_row<D, CT>(p.v_pool, row, l, v0, v1);
    if (l == 0) *reinterpret_cast<f32x2*>(p.scales + row * 2) = s;
}

template <typename T, int D, int CT>
__global__ __launch_bounds__(kRowThreads) void read_kernel(RowsParams p, void* k_out, void* v_out) {
    int r, hk, l;
    if (!row_of<D / 8>(p, r, hk, l)) return;
    const int slot = p.slots[r];
    if (slot < 0) return;
    const size_t row = pool_row(p, slot, hk), from = row * D + 8 * l, to = ((size_t)r * p.Hkv + hk) * D + 8 * l;
    float a[8], b[8];
    if constexpr (CT == kCacheF16) {
        load8<_Float16>(p.k_pool, from, a);
        load8<_Float16>(p.v_pool, from, b);
    } else {
        const u32x2 ck = *reinterpret_cast<const u32x2*>(static_cast<const unsigned char*>(p.k_pool) + from);
        const u32x2 cv = *reinterpret_cast<const u32x2*>(static_cast<const unsigned char*>(p.v_pool) + from);
        const f32x2 s = *reinterpret_cast<const f32x2*>(p.scales + row * 2);
        const f16x8 x = codes_to_f16x8<CT>(ck), y = codes_to_f16x8<CT>(cv);
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = (float)x[e] * s[0], b[e] = (float)y[e] * s[1];
    }
    store8<T>(k_out, to, a);
    store8<T>(v_out, to, b);
}

template <typename F>
int for_head_dim(int D, F&& f) {
    switch (D) {
        case 32: return f(std::integral_constant<int, 32>{});
        case 64: return f(std::integral_constant<int, 64>{});
        case 128: return f(std::integral_constant<int, 128>{});
        case 256: return f(std::integral_constant<int, 256>{});
        default: return set_error(KVC_ERR_UNSUPPORTED, "head_dim must be 32, 64, 128 or 256");
    }
}

template <typename F>
int guard_rows(F&& f) {
    try {
        return f();
    } catch (...) {
        return set_error(KVC_ERR_STATE, "unexpected exception");
    }
}

unsigned row_groups(int rows, int Hkv, int lanes) {
    const int per = kRowThreads / lanes;
    return (unsigned)((rows + (long long)per - 1) / per * Hkv);
}

bool a16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// What the three entry points share: shape, the cache's type and its pointers.
int check_cache(int rows, int Hkv, int D, int BLOCK, int kv_dtype, bool f16_ok, const void* k_pool, const void* v_pool,
                const void* scales, const int* slots) {
    if (kv_dtype == KVC_F32 || (kv_dtype == KVC_F16 && !f16_ok))
        return set_error(KVC_ERR_UNSUPPORTED, f16_ok ? "the cache must be KVC_F16, KVC_I8 or KVC_E4M3"
                                                     : "the cache must be KVC_I8 or KVC_E4M3 (kvc_write_kv_slots "
                                                       "writes KVC_F16)");
    if (kv_dtype != KVC_F16 && kv_dtype != KVC_I8 && kv_dtype != KVC_E4M3)
        return set_error(KVC_ERR_ARG, "kv_dtype must be KVC_F16, KVC_I8 or KVC_E4M3");
    if (rows < 0 || Hkv <= 0 || BLOCK <= 0) return set_error(KVC_ERR_ARG, "rows must be >= 0, Hkv and BLOCK > 0");
    if (D != 32 && D != 64 && D != 128 && D != 256)
        return set_error(KVC_ERR_UNSUPPORTED, "head_dim must be 32, 64, 128 or 256");
    if ((long long)rows * 2 * Hkv >= 1LL << 31) return set_error(KVC_ERR_UNSUPPORTED, "rows * 2 * Hkv must be below 2^31");
    if (rows == 0) return KVC_OK;
    if (!k_pool || !v_pool || !slots) return set_error(KVC_ERR_ARG, "null pool or slot pointer");
    if (!a16(k_pool) || !a16(v_pool)) return set_error(KVC_ERR_ARG, "the pools must be 16-byte aligned");
    if (kv_dtype != KVC_F16 && (!scales || ((uintptr_t)scales & 7u)))
        return set_error(KVC_ERR_ARG, "an 8-bit cache needs its scales, 8-byte aligned");
    return KVC_OK;
}

}  // namespace
}  // namespace kvc

using namespace kvc;

extern "C" {

int kvc_qk_norm_rope_write(void* q, void* k_pool, void* v_pool, float* kv_scales, const void* qkv, long long row_stride,
                           const int* pos, const int* slots, const void* q_norm, const void* k_norm, float eps,
                           float theta, int M, int Hq, int Hkv, int D, int BLOCK, int kv_dtype, kvc_stream_t st) {
    return guard_rows([&]() -> int {
        int rc = check_cache(M, Hkv, D, BLOCK, kv_dtype, true, k_pool, v_pool, kv_scales, slots);
        if (rc) return rc;
        if (Hq <= 0 || Hq % Hkv) return set_error(KVC_ERR_ARG, "Hq must be a positive multiple of Hkv");
        if (Hq + 2LL * Hkv > 1 << 16) return set_error(KVC_ERR_UNSUPPORTED, "at most 65536 heads");
        if (!(eps >= 0.f) || !(theta > 1.f) || !std::isfinite(theta) || !std::isfinite(eps))
            return set_error(KVC_ERR_ARG, "eps must be >= 0 and theta > 1, both finite");
        const long long width = ((long long)Hq + 2LL * Hkv) * D;
        if (row_stride == 0) row_stride = width;
        if (row_stride < width || row_stride % 8)
            return set_error(KVC_ERR_ARG, "row_stride must be a multiple of 8 of at least (Hq + 2 Hkv) * D elements");
        if (M == 0) return KVC_OK;
        if (!q || !qkv || !pos || q == qkv) return set_error(KVC_ERR_ARG, "null q, qkv or pos, or q is qkv");
        if (!a16(q) || !a16(qkv) || !a16(q_norm) || !a16(k_norm))
            return set_error(KVC_ERR_ARG, "q, qkv and the norm weights must be 16-byte aligned");
        RopeWriteParams p{static_cast<_Float16*>(q), k_pool, v_pool, kv_scales, static_cast<const _Float16*>(qkv),
                          row_stride, pos, slots, static_cast<const _Float16*>(q_norm),
                          static_cast<const _Float16*>(k_norm), eps, std::log2((double)theta), M, Hq, Hkv, BLOCK, 1};
        return for_head_dim(D, [&](auto d) -> int {
            constexpr int kD = decltype(d)::value;
            const dim3 grid((unsigned)((M + p.tokens - 1) / p.tokens));
            const size_t lds = (size_t)p.tokens * (kD / 2) * sizeof(f32x2);
            if (kv_dtype == KVC_F16)
                hipLaunchKernelGGL((norm_rope_write_kernel<kD, kCacheF16>), grid, dim3(kRowThreads), lds, (hipStream_t)st, p);
            else if (kv_dtype == KVC_I8)
                hipLaunchKernelGGL((norm_rope_write_kernel<kD, kCacheI8>), grid, dim3(kRowThreads), lds, (hipStream_t)st, p);
            else
                hipLaunchKernelGGL((norm_rope_write_kernel<kD, kCacheE4M3>), grid, dim3(kRowThreads), lds, (hipStream_t)st, p);
            return hip_check(hipGetLastError(), "norm, rotary and cache write launch");
        });
    });
}

int kvc_write_kv_q8(const void* k, const void* v, void* k_pool, void* v_pool, float* kv_scales, const int* slot_map,
                    int rows, int Hkv, int D, int BLOCK, int dtype, int kv_dtype, kvc_stream_t st) {
    return guard_rows([&]() -> int {
        int rc = check_cache(rows, Hkv, D, BLOCK, kv_dtype, false, k_pool, v_pool, kv_scales, slot_map);
        if (rc) return rc;
        if (dtype != KVC_F16 && dtype != KVC_F32) return set_error(KVC_ERR_ARG, "dtype must be KVC_F32 (0) or KVC_F16 (1)");
        if (rows == 0) return KVC_OK;
        if (!k || !v || !a16(k) || !a16(v)) return set_error(KVC_ERR_ARG, "k and v must be 16-byte aligned and not null");
        const RowsParams p{k, v, k_pool, v_pool, kv_scales, slot_map, rows, Hkv, BLOCK};
        return for_head_dim(D, [&](auto d) -> int {
            constexpr int kD = decltype(d)::value;
            const dim3 grid(row_groups(rows, Hkv, kD / 16)), block(kRowThreads);
            const hipStream_t s = (hipStream_t)st;
            if (dtype == KVC_F16 && kv_dtype == KVC_I8)
                hipLaunchKernelGGL((write_q8_kernel<_Float16, kD, kCacheI8>), grid, block, 0, s, p);
            else if (dtype == KVC_F16)
                hipLaunchKernelGGL((write_q8_kernel<_Float16, kD, kCacheE4M3>), grid, block, 0, s, p);
            else if (kv_dtype == KVC_I8)
                hipLaunchKernelGGL((write_q8_kernel<float, kD, kCacheI8>), grid, block, 0, s, p);
            else
                hipLaunchKernelGGL((write_q8_kernel<float, kD, kCacheE4M3>), grid, block, 0, s, p);
            return hip_check(hipGetLastError(), "quantised kv write launch");
        });
    });
}

int kvc_read_kv(void* k, void* v, const void* k_pool, const void* v_pool, const float* kv_scales, const int* slot_map,
                int rows, int Hkv, int D, int BLOCK, int dtype, int kv_dtype, kvc_stream_t st) {
    return guard_rows([&]() -> int {
        int rc = check_cache(rows, Hkv, D, BLOCK, kv_dtype, true, k_pool, v_pool, kv_scales, slot_map);
        if (rc) return rc;
        if (dtype != KVC_F16 && dtype != KVC_F32) return set_error(KVC_ERR_ARG, "dtype must be KVC_F32 (0) or KVC_F16 (1)");
        if (rows == 0) return KVC_OK;
        if (!k || !v || !a16(k) || !a16(v)) return set_error(KVC_ERR_ARG, "k and v must be 16-byte aligned and not null");
        const RowsParams p{nullptr, nullptr, const_cast<void*>(k_pool), const_cast<void*>(v_pool),
                           const_cast<float*>(kv_scales), slot_map, rows, Hkv, BLOCK};
        return for_head_dim(D, [&](auto d) -> int {
            constexpr int kD = decltype(d)::value;
            const dim3 grid(row_groups(rows, Hkv, kD / 8)), block(kRowThreads);
            const hipStream_t s = (hipStream_t)st;
            auto launch = [&](auto ct) {
                constexpr int kCT = decltype(ct)::value;
                if (dtype == KVC_F16) hipLaunchKernelGGL((read_kernel<_Float16, kD, kCT>), grid, block, 0, s, p, k, v);
                else hipLaunchKernelGGL((read_kernel<float, kD, kCT>), grid, block, 0, s, p, k, v);
            };
            if (kv_dtype == KVC_F16) launch(std::integral_constant<int, kCacheF16>{});
            else if (kv_dtype == KVC_I8) launch(std::integral_constant<int, kCacheI8>{});
            else launch(std::integral_constant<int, kCacheE4M3>{});
            return hip_check(hipGetLastError(), "kv read launch");
        });
    });
}

}  // extern "C"
