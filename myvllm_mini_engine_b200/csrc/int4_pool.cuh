// The 4-bit KV pool: its page format, and the kernels that write and read rows.
//
// Format.  A pool is [num_blocks, kv_heads, page_bytes] bytes.  The page of one
// kv head is contiguous: block_size rows of D/2 bytes (element 2i in the low
// half of byte i), then block_size pairs of fp16 (step, base), padded to 16
// bytes.  An element reads as base + step * code, code in 0..15; a stored step
// below 2^-24 reads as 2^-24.  A row (one token, one kv head, K or V) is
// quantised by itself: base = fp16(min), step = fp16(max(2^-24, (max - min) / 15)),
// code = round((x - base) / step) clamped to 0..15 (true quotients, nearest
// even).  NaN counts as 0 and magnitudes saturate at 65504.  At D = 128 a row
// takes 68 bytes, 4.25 bits an element, against 256 in a 16-bit pool.  One
// pair per row (not per smaller group) lets the attention fold the key's step
// into the score and the value's step into the probability, so that the codes
// go into the matrix instructions as they are.  The page is head-major so that
// a kv head's part of a page is one run: a warp that attends one kv head reads
// 1 KB runs at D = 128, block_size 16.
#pragma once

#include "common.cuh"
#include "row_maps.cuh"

namespace minikv {

__host__ __device__ constexpr int64_t int4_page_bytes(int64_t block_size, int64_t head_dim) {
    return (block_size * (head_dim / 2 + 4) + 15) / 16 * 16;
}

constexpr float kInt4StepMin = 1.f / 16777216.f;  // 2^-24, the smallest fp16

// Lanes that share a row in the row kernels: 8 elements a lane, a power of two.
constexpr int int4_row_lanes(int D) { return D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// 8 consecutive elements at p as fp32.  VEC: p is 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const T* p, float* f) {
    if constexpr (VEC) {
        constexpr int n = 8 / Elem<T>::kPerVec;
#pragma unroll
        for (int i = 0; i < n; ++i)
            Elem<T>::load(ld_global_nc(reinterpret_cast<const uint4*>(p) + i), f + i * Elem<T>::kPerVec);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = Elem<T>::to_float(p[i]);
    }
}

// Quantising write.  A unit is one row: (token, kv head, K or V); a group of
// int4_row_lanes(D) lanes takes one, 8 elements a lane, so at D = 128 a warp
// takes the K and the V row of a token's head.  Bound by the bytes of the
// 16-bit rows it reads.
template <typename T, int D, bool VEC, typename Rows>
__global__ void __launch_bounds__(256) int4_write_kernel(
    unsigned char* __restrict__ kc, unsigned char* __restrict__ vc, const T* __restrict__ k, const T* __restrict__ v,
    int64_t tokens, int kv_heads, int64_t block_size, int64_t page_bytes, int64_t k_stride, int64_t v_stride,
    Rows map) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int LPR = int4_row_lanes(D);
    const int sub = threadIdx.x % LPR;
    const bool active = sub * 8 < D;
    const int64_t units = tokens * kv_heads * 2;
    const int64_t groups = (int64_t)gridDim.x * (blockDim.x / LPR);
    // units of a block are consecutive; the loop bound is the same for a whole warp (the shuffles need all lanes)
    const int64_t first = (int64_t)blockIdx.x * (blockDim.x / LPR) + threadIdx.x / LPR;
    const int64_t warp_first = first - (threadIdx.x % 32) / LPR;
    for (int64_t off = 0; warp_first + off < units; off += groups) {
        const int64_t u = first + off;
        const bool in = u < units;
        const int64_t t = in ? u / (2 * kv_heads) : 0;
        const int rest = in ? (int)(u - t * (2 * kv_heads)) : 0;
        const int h = rest >> 1, which = rest & 1;
        const int64_t row = in ? map(t) : -1;
        float x[8];
        float lo = INFINITY, hi = -INFINITY;
        if (row >= 0 && active) {
            load_row8<T, VEC>((which ? v + t * v_stride : k + t * k_stride) + (int64_t)h * D + sub * 8, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = isnan(x[i]) ? 0.f : fminf(fmaxf(x[i], -65504.f), 65504.f);
                lo = fminf(lo, x[i]);
                hi = fmaxf(hi, x[i]);
            }
        }
#pragma unroll
        for (int m = LPR / 2; m > 0; m >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
        }
        if (row < 0) continue;  // no shuffle follows in this iteration
        const __half base = __float2half_rn(lo);
        const __half step = __float2half_rn(fmaxf(__fdiv_rn(hi - lo, 15.f), kInt4StepMin));
        const float b = __half2float(base), s = __half2float(step), inv = __fdiv_rn(1.f, s);
        const int64_t page = row / block_size, off_in = row - page * block_size;
        unsigned char* dst = (which ? vc : kc) + (page * kv_heads + h) * page_bytes;
        if (active) {
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = x[i] - b;
                const float q = d * inv;  // within 2e-6 of the quotient where that lies in 0..15
                float c = rintf(q);
                // next to a half: the true quotient decides.  Rare, so the division stays off the common path
                if (fabsf(fabsf(q - c) - 0.5f) < 1e-4f) c = rintf(__fdiv_rn(d, s));
                word |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * i);
            }
            *reinterpret_cast<uint32_t*>(dst + off_in * (D / 2) + sub * 4) = word;
        }
        if (sub == 0)
            *reinterpret_cast<__half2*>(dst + block_size * (D / 2) + off_in * 4) = __halves2half2(step, base);
    }
}

// Reading rows back: out[t] = the values of slot t (zeros for a slot outside the pool).
template <typename T, int D>
__global__ void __launch_bounds__(256) int4_read_kernel(
    const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc, T* __restrict__ k, T* __restrict__ v,
    int64_t tokens, int kv_heads, int64_t block_size, int64_t page_bytes, SlotRows map) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int LPR = int4_row_lanes(D);
    const int sub = threadIdx.x % LPR;
    if (sub * 8 >= D) return;
    const int64_t units = tokens * kv_heads * 2;
    const int64_t groups = (int64_t)gridDim.x * (blockDim.x / LPR);
    for (int64_t u = (int64_t)blockIdx.x * (blockDim.x / LPR) + threadIdx.x / LPR; u < units; u += groups) {
        const int64_t t = u / (2 * kv_heads);
        const int rest = (int)(u - t * (2 * kv_heads));
        const int h = rest >> 1, which = rest & 1;
        const int64_t row = map(t);
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (row >= 0) {
            const int64_t page = row / block_size, off_in = row - page * block_size;
            const unsigned char* src = (which ? vc : kc) + (page * kv_heads + h) * page_bytes;
            const uint32_t word = *reinterpret_cast<const uint32_t*>(src + off_in * (D / 2) + sub * 4);
            const float2 sb =
                __half22float2(*reinterpret_cast<const __half2*>(src + block_size * (D / 2) + off_in * 4));
            const float s = fmaxf(sb.x, kInt4StepMin);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __fadd_rn(sb.y, __fmul_rn(s, (float)((word >> (4 * i)) & 15u)));
        }
        uint4* dst = reinterpret_cast<uint4*>((which ? v : k) + (t * kv_heads + h) * D + sub * 8);
#pragma unroll
        for (int i = 0; i < 8 / Elem<T>::kPerVec; ++i) dst[i] = Elem<T>::store(x + i * Elem<T>::kPerVec);
    }
}

// Blocks of 256 threads for `units` rows of `lanes` lanes each, at most 8 a SM.
inline unsigned int4_grid(int64_t units, int lanes, int sms) {
    const int64_t per = 256 / lanes, blocks = (units + per - 1) / per, cap = (int64_t)sms * 8;
    return (unsigned)(blocks < 1 ? 1 : blocks < cap ? blocks : cap);
}

template <typename T, int D, typename Rows>
static cudaError_t launch_int4_write(void* kc, void* vc, const void* k, const void* v, int64_t tokens, int kv_heads,
                                     int64_t block_size, int64_t k_stride, int64_t v_stride, bool vec, Rows map,
                                     int sms, cudaStream_t stream) {
    return launch_chained(vec ? int4_write_kernel<T, D, true, Rows> : int4_write_kernel<T, D, false, Rows>,
                          dim3(int4_grid(tokens * kv_heads * 2, int4_row_lanes(D), sms)), dim3(256), 0, stream,
                          static_cast<unsigned char*>(kc), static_cast<unsigned char*>(vc), static_cast<const T*>(k),
                          static_cast<const T*>(v), tokens, kv_heads, block_size, int4_page_bytes(block_size, D),
                          k_stride, v_stride, map);
}

template <typename T, int D>
static cudaError_t launch_int4_read(const void* kc, const void* vc, void* k, void* v, int64_t tokens, int kv_heads,
                                    int64_t block_size, SlotRows map, int sms, cudaStream_t stream) {
    return launch_chained(int4_read_kernel<T, D>, dim3(int4_grid(tokens * kv_heads * 2, int4_row_lanes(D), sms)),
                          dim3(256), 0, stream, static_cast<const unsigned char*>(kc),
                          static_cast<const unsigned char*>(vc), static_cast<T*>(k), static_cast<T*>(v), tokens,
                          kv_heads, block_size, int4_page_bytes(block_size, D), map);
}

}  // namespace minikv
