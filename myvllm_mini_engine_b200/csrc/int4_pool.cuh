// The 4-bit KV pool: its page format, and the kernels that write and read rows.
//
// Format.  A pool is [num_blocks, kv_heads, page_bytes] bytes.  The page of one
// kv head is contiguous: block_size rows of D/2 bytes (element 2i in the low
// half of byte i), then block_size pairs of fp16 (step, base), padded to 16
// bytes.  An element reads as base + step * code, code in 0..15; a stored step
// below 2^-24 reads as 2^-24.  A row (one token, one kv head, K or V) is
// quantised by itself: base = fp16(min), step = fp16(max(2^-24, (max - min) / 15)),
// code = round((x - base) / step) clamped to 0..15 (true quotients, nearest
// even).  NaN counts as 0 and magnitudes saturate at 65504; where base + 15 step
// would pass it, the step is the largest fp16 with which it does not (2^-24 at
// least): every element then reads as a finite fp16.  At D = 128 a row
// takes 68 bytes, 4.25 bits an element, against 256 in a 16-bit pool.  One
// pair per row (not per smaller group) lets the attention fold the key's step
// into the score and the value's step into the probability, so that the codes
// go into the matrix instructions as they are.  The page is head-major so that
// a kv head's part of a page is one run: a warp that attends one kv head reads
// 1 KB runs at D = 128, block_size 16.
#pragma once

#include <string.h>

#include <type_traits>

#include "common.cuh"
#include "row_maps.cuh"

namespace minikv {

__host__ __device__ constexpr int64_t int4_page_bytes(int64_t block_size, int64_t head_dim) {
    return (block_size * (head_dim / 2 + 4) + 15) / 16 * 16;
}

// n / d for n < 2^31: a product and a shift.
struct FastDiv {
    uint32_t d, m, s;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor), s(0) {
        while ((1ull << s) < divisor) ++s;
        m = (uint32_t)((((1ull << s) - divisor) << 32) / divisor + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

constexpr float kInt4StepMin = 1.f / 16777216.f;  // 2^-24, the smallest fp16

// Blocks of 256 threads a SM in the row kernels: the grid fills the device once.
constexpr int kInt4WriteBlocks = 4, kInt4ReadBlocks = 5;

// Lanes that share a row of D elements, E each: a power of two.
constexpr int int4_row_lanes(int D, int E = 8) { return D / E <= 2 ? 2 : D / E <= 4 ? 4 : D / E <= 8 ? 8 : D / E <= 16 ? 16 : 32; }

// 16 consecutive elements of a row, held as they came.  VEC: p is 16-byte aligned.
template <typename T, bool VEC> struct RowPart {
    static constexpr int VECS = 16 / Elem<T>::kPerVec;
    uint4 v[VECS];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < VECS; ++i) {
            if constexpr (VEC) {
                v[i] = ld_global_nc(reinterpret_cast<const uint4*>(p) + i);
            } else {
                T x[Elem<T>::kPerVec];
#pragma unroll
                for (int e = 0; e < Elem<T>::kPerVec; ++e) x[e] = p[i * Elem<T>::kPerVec + e];
                memcpy(&v[i], x, 16);
            }
        }
    }
    // Least and largest of the 16, and whether one is NaN, infinite or over 65504 in magnitude.
    __device__ __forceinline__ bool extremes(const float* f, float* lo, float* hi) const {
        bool odd;
        if constexpr (sizeof(T) == 2) {  // two elements an operation
            using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            const Pair* x = reinterpret_cast<const Pair*>(v);
            const uint32_t zero = 0u;
            Pair l = x[0], h = x[0], bad = __hmul2(x[0], *reinterpret_cast<const Pair*>(&zero));
#pragma unroll
            for (int i = 1; i < 8; ++i) {
                l = __hmin2(l, x[i]);
                h = __hmax2(h, x[i]);
                bad = __hfma2(x[i], *reinterpret_cast<const Pair*>(&zero), bad);
            }
            float a[2], b[2];
            Elem<T>::unpack(*reinterpret_cast<uint32_t*>(&l), a);
            Elem<T>::unpack(*reinterpret_cast<uint32_t*>(&h), b);
            *lo = fminf(a[0], a[1]);
            *hi = fmaxf(b[0], b[1]);
            odd = (*reinterpret_cast<uint32_t*>(&bad) & 0x7fff7fffu) != 0u;  // NaN from NaN and infinities
        } else {
            float bad = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                *lo = fminf(*lo, f[i]);
                *hi = fmaxf(*hi, f[i]);
                bad = fmaf(f[i], 0.f, bad);
            }
            odd = !(bad == 0.f);
        }
        return odd || *lo < -65504.f || *hi > 65504.f;
    }
    __device__ __forceinline__ void values(float* f) const {
#pragma unroll
        for (int i = 0; i < VECS; ++i) Elem<T>::load(v[i], f + i * Elem<T>::kPerVec);
    }
};

// The step of a row from lo to hi whose base is b.
__device__ __forceinline__ __half int4_step(float lo, float hi, float b) {
    __half step = __float2half_rn(fmaxf(__fdiv_rn(hi - lo, 15.f), kInt4StepMin));
    if (__fadd_rn(b, 15.f * __half2float(step)) > 65504.f)  // rare: rows that end near 65504
        step = __float2half_rd(fmaxf(__fdiv_rd(__fsub_rd(65504.f, b), 15.f), kInt4StepMin));
    return step;
}

// Code of one element by the format's own words.
__device__ __forceinline__ uint32_t int4_code(float x, float base, float step) {
    return (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(x - base, step)), 0.f), 15.f);
}

// Quantising write.  A unit is one row: (token, kv head, K or V); a group of
// int4_row_lanes(D, 16) lanes takes one, 16 elements a lane, so at D = 128 a
// warp takes the K and the V rows of two heads of a token (8 elements a lane,
// twice the row's own work an element, took a third longer).  Bound by issue: 75 %
// of the slots used; 16384 tokens of 8 heads of 128 in fp16 28.7 us, 3.0 TB/s.  The usual row costs an
// element a subtraction, two products with the rounded inverse of the step (a
// little above and a little below it, each rounded to a whole number by an
// addition of 1.5 2^23) and an addition into the word: where the two agree, so
// does the true quotient.  Where they differ, and for rows with NaN, infinities,
// magnitudes above 65504 or codes to clamp, the lane divides.
template <typename T, int D, bool VEC, typename Rows>
__global__ void __launch_bounds__(256, kInt4WriteBlocks) int4_write_kernel(
    unsigned char* __restrict__ kc, unsigned char* __restrict__ vc, const T* __restrict__ k, const T* __restrict__ v,
    int64_t first_token, int64_t tokens, int kv_heads, FastDiv rows_of, FastDiv block_of, int64_t page_bytes,
    int64_t k_stride, int64_t v_stride, Rows map) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int LPR = int4_row_lanes(D, 16);
    constexpr float kRound = 12582912.f;  // 1.5 2^23
    const int sub = threadIdx.x % LPR;
    const bool active = sub * 16 < D;
    const uint32_t units = (uint32_t)(tokens * kv_heads * 2);
    const uint32_t groups = gridDim.x * (blockDim.x / LPR);
    // the loop's bound is the same for a whole warp: the shuffles need all lanes
    const uint32_t first = blockIdx.x * (blockDim.x / LPR) + threadIdx.x / LPR;
    const uint32_t warp_first = first - (threadIdx.x % 32) / LPR;
    struct Unit {
        int64_t token;
        uint32_t h;
        bool in, which;
    };
    auto unit_at = [&](uint32_t u) {
        const bool in = u < units;
        const uint32_t t = rows_of(in ? u : 0), rest = in ? u - t * rows_of.d : 0;
        return Unit{first_token + t, rest >> 1, in, (rest & 1) != 0};
    };
    auto source = [&](const Unit& n) {
        return (n.which ? v + n.token * v_stride : k + n.token * k_stride) + (int64_t)n.h * D + sub * 16;
    };
    RowPart<T, VEC> ahead;  // the next row, loaded while this one is worked on
    Unit next = unit_at(first);
    if (active) ahead.load(source(next));
    for (uint32_t off = 0; warp_first + off < units; off += groups) {
        const Unit n = next;
        const RowPart<T, VEC> raw = ahead;
        const int64_t row = n.in ? map(n.token) : -1;
        if (warp_first + off + groups < units) {
            next = unit_at(first + off + groups);
            if (active) ahead.load(source(next));
        }
        const uint32_t h = n.h;
        const bool which = n.which;
        float x[16];
        float lo = INFINITY, hi = -INFINITY;
        if (active) {
            raw.values(x);
            const bool odd = raw.extremes(x, &lo, &hi);
            if (odd) {
                lo = INFINITY;
                hi = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    x[i] = isnan(x[i]) ? 0.f : fminf(fmaxf(x[i], -65504.f), 65504.f);
                    lo = fminf(lo, x[i]);
                    hi = fmaxf(hi, x[i]);
                }
            }
        }
#pragma unroll
        for (int m = LPR / 2; m > 0; m >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
        }
        if (row < 0) continue;  // no shuffle follows in this iteration
        const __half base = __float2half_rn(lo);
        const float b = __half2float(base);
        const __half step = int4_step(lo, hi, b);
        const float s = __half2float(step);
        float inv;  // 1 / s within 2^-22
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
        const uint32_t page = block_of((uint32_t)row), off_in = (uint32_t)row - page * block_of.d;
        unsigned char* dst = (which ? vc : kc) + ((int64_t)page * kv_heads + h) * page_bytes;
        if (active) {
            const float over = inv * (1.f + 1.f / 1048576.f), under = inv * (1.f - 1.f / 1048576.f);
            uint32_t word[2] = {0u, 0u}, differ = 0;
            bool clamp = (lo - b) * inv < -0.49f || (hi - b) * inv > 15.49f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float d = x[i] - b;
                const uint32_t up = __float_as_uint(fmaf(d, over, kRound)), down = __float_as_uint(fmaf(d, under, kRound));
                differ |= up ^ down;
                word[i / 8] += up << (4 * (i % 8));  // 0x4b400000 + code, the constants taken out below
            }
            word[0] -= 0x3f400000u;  // 0x4b400000 (1 + 2^4 + 2^8 + ...) mod 2^32
            word[1] -= 0x3f400000u;
            if (differ != 0 || clamp) {
                word[0] = word[1] = 0u;
#pragma unroll
                for (int i = 0; i < 16; ++i) word[i / 8] |= int4_code(x[i], b, s) << (4 * (i % 8));
            }
            *reinterpret_cast<uint2*>(dst + (int64_t)off_in * (D / 2) + sub * 8) = make_uint2(word[0], word[1]);
        }
        if (sub == 0)
            *reinterpret_cast<__half2*>(dst + (int64_t)block_of.d * (D / 2) + (int64_t)off_in * 4) =
                __halves2half2(step, base);
    }
}

// Reading rows back: out[t] = the values of slot t (zeros for a slot outside the pool).
template <typename T, int D>
__global__ void __launch_bounds__(256, kInt4ReadBlocks) int4_read_kernel(
    const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc, T* __restrict__ k, T* __restrict__ v,
    int64_t first_token, int64_t tokens, int kv_heads, FastDiv rows_of, FastDiv block_of, int64_t page_bytes,
    SlotRows map) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int LPR = int4_row_lanes(D);
    const int sub = threadIdx.x % LPR;
    if (sub * 8 >= D) return;
    const uint32_t units = (uint32_t)(tokens * kv_heads * 2);
    const uint32_t groups = gridDim.x * (blockDim.x / LPR);
#pragma unroll 4
    for (uint32_t u = blockIdx.x * (blockDim.x / LPR) + threadIdx.x / LPR; u < units; u += groups) {
        const uint32_t t = rows_of(u);
        const uint32_t rest = u - t * rows_of.d, h = rest >> 1;
        const bool which = rest & 1;
        const int64_t token = first_token + t;
        const int64_t row = map(token);
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (row >= 0) {
            const uint32_t page = block_of((uint32_t)row), off_in = (uint32_t)row - page * block_of.d;
            const unsigned char* src = (which ? vc : kc) + ((int64_t)page * kv_heads + h) * page_bytes;
            const uint32_t word = *reinterpret_cast<const uint32_t*>(src + (int64_t)off_in * (D / 2) + sub * 4);
            const float2 sb = __half22float2(*reinterpret_cast<const __half2*>(
                src + (int64_t)block_of.d * (D / 2) + (int64_t)off_in * 4));
            const float s = fmaxf(sb.x, kInt4StepMin);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __fadd_rn(sb.y, __fmul_rn(s, (float)((word >> (4 * i)) & 15u)));
        }
        uint4* dst = reinterpret_cast<uint4*>((which ? v : k) + (token * kv_heads + h) * D + sub * 8);
#pragma unroll
        for (int i = 0; i < 8 / Elem<T>::kPerVec; ++i) dst[i] = Elem<T>::store(x + i * Elem<T>::kPerVec);
    }
}

// Blocks of 256 threads for `units` rows of `lanes` lanes each, at most those that run at once.
inline unsigned int4_grid(int64_t units, int lanes, int blocks_a_sm, int sms) {
    const int64_t per = 256 / lanes, blocks = (units + per - 1) / per, cap = (int64_t)sms * blocks_a_sm;
    return (unsigned)(blocks < 1 ? 1 : blocks < cap ? blocks : cap);
}

// Tokens of a launch: its rows are counted in 31 bits.
inline int64_t int4_tokens_at_once(int kv_heads) { return (1ll << 30) / kv_heads; }

template <typename T, int D, typename Rows>
static cudaError_t launch_int4_write(void* kc, void* vc, const void* k, const void* v, int64_t tokens, int kv_heads,
                                     int64_t block_size, int64_t k_stride, int64_t v_stride, bool vec, Rows map,
                                     int sms, cudaStream_t stream) {
    const int64_t most = int4_tokens_at_once(kv_heads) - 1;
    cudaError_t err = cudaSuccess;
    for (int64_t t = 0; t < tokens && err == cudaSuccess; t += most) {
        const int64_t n = tokens - t < most ? tokens - t : most;
        err = launch_chained(vec ? int4_write_kernel<T, D, true, Rows> : int4_write_kernel<T, D, false, Rows>,
                             dim3(int4_grid(n * kv_heads * 2, int4_row_lanes(D, 16), kInt4WriteBlocks, sms)), dim3(256), 0,
                             stream, static_cast<unsigned char*>(kc), static_cast<unsigned char*>(vc),
                             static_cast<const T*>(k), static_cast<const T*>(v), t, n, kv_heads,
                             FastDiv((uint32_t)kv_heads * 2), FastDiv((uint32_t)block_size),
                             int4_page_bytes(block_size, D), k_stride, v_stride, map);
    }
    return err;
}

template <typename T, int D>
static cudaError_t launch_int4_read(const void* kc, const void* vc, void* k, void* v, int64_t tokens, int kv_heads,
                                    int64_t block_size, SlotRows map, int sms, cudaStream_t stream) {
    const int64_t most = int4_tokens_at_once(kv_heads) - 1;
    cudaError_t err = cudaSuccess;
    for (int64_t t = 0; t < tokens && err == cudaSuccess; t += most) {
        const int64_t n = tokens - t < most ? tokens - t : most;
        err = launch_chained(int4_read_kernel<T, D>, dim3(int4_grid(n * kv_heads * 2, int4_row_lanes(D), kInt4ReadBlocks, sms)),
                             dim3(256), 0, stream, static_cast<const unsigned char*>(kc),
                             static_cast<const unsigned char*>(vc), static_cast<T*>(k), static_cast<T*>(v), t, n,
                             kv_heads, FastDiv((uint32_t)kv_heads * 2), FastDiv((uint32_t)block_size),
                             int4_page_bytes(block_size, D), map);
    }
    return err;
}

}  // namespace minikv
