// Selecting the blocks a query attends: key bounds of every block, and the
// blocks of highest score.
//
// Bounds.  [num_blocks, kv_heads, 2 D + 16] bytes: D int8 codes of the keys'
// elementwise maximum over the block's rows, D of their minimum, one fp32 scale
// (12 bytes of padding).  scale = top / 127 with top the largest magnitude of
// the 2 D bounds; codes ceil(127 max / top) and floor(127 min / top), so that
// code * scale bounds the keys, but for the two fp32 roundings of scale and
// product (2^-23 of the bound).  A block whose top is below 2^-100 has zero
// codes and scale.  NaN keys count as 0, infinite ones as the largest fp32.
//
// Score.  For a kv head with query heads q_1 .. q_n, let qp = sum_h max(q_h, 0)
// and qn = sum_h min(q_h, 0) (fp32, in the order of the heads).  Then for any
// key k of the block, sum_h q_h . k <= sum_d max_d qp_d + min_d qn_d.  The 2 D
// values (qp, qn) are held in 8 bits over their largest magnitude, a factor
// common to all blocks of the kv head, so
//   score = scale_block * (sum_d maxcode_d qpcode_d + mincode_d qncode_d)
// where the sum is a whole number below 2^24: it has one value whatever the
// order, and with it the selection.  (The codes are rounded to nearest: a score
// stands for the bound up to half a code of each, and is not itself one.)
// 8-bit bounds are a sixteenth of the bytes of a 16-bit block of 16 tokens (K and
// V: 64 D bytes), and an eighth of those of a 4-bit one.
#pragma once

#include <string.h>

#include "common.cuh"
#include "int4_pool.cuh"

namespace minikv {

constexpr int kBoundsPad = 16;
constexpr float kBoundsNone = 7.8886090522101181e-31f;  // 2^-100
constexpr float kLargest = 3.4028234663852886e+38f;

// ------------------------------------------------------------ key rows
// E consecutive elements (1, 2, 4 or 8) of dims (i * 32 + lane) * E of a row, as fp32.
template <typename T, int E> struct RowElems {  // 16-bit or fp32 pool
    __device__ static __forceinline__ void load(const T* row, int d, float* f) {
        if constexpr (sizeof(T) * E == 16) {
            Elem<T>::load(*reinterpret_cast<const uint4*>(row + d), f);
        } else if constexpr (sizeof(T) * E == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(row + d);
            if constexpr (sizeof(T) == 4) {
                f[0] = __uint_as_float(v.x);
                f[1] = __uint_as_float(v.y);
            } else {
                Elem<T>::unpack(v.x, f);
                Elem<T>::unpack(v.y, f + 2);
            }
        } else if constexpr (sizeof(T) * E == 4 && sizeof(T) == 2) {
            Elem<T>::unpack(*reinterpret_cast<const uint32_t*>(row + d), f);
        } else {
            f[0] = Elem<T>::to_float(row[d]);
        }
    }
};

// Elements a lane takes at once: a warp's 32 lanes cover 32 E dims of the D.
template <typename T> constexpr int bounds_elems(int D) {
    const int most = 16 / (int)sizeof(T);
    const int per = D / 32;
    return per % 8 == 0 && most >= 8 ? 8 : per % 4 == 0 && most >= 4 ? 4 : per % 2 == 0 ? 2 : 1;
}
struct Int4Tag {};
template <> constexpr int bounds_elems<Int4Tag>(int D) {
    const int per = D / 32;
    return per % 8 == 0 ? 8 : per % 4 == 0 ? 4 : per % 2 == 0 ? 2 : 1;
}

// ceil (UP) or floor of 127 x / top, exactly: an fp32 estimate (within 2e-5), and next to a whole
// number the products in 64 bits, which hold them exactly.
template <bool UP> __device__ __forceinline__ int bound_code(float x, float top, float inv) {
    const float t = x * inv;
    const float k = rintf(t);
    int c;
    if (fabsf(t - k) < 1e-3f) {
        const double a = 127.0 * (double)x, b = (double)k * (double)top;
        c = (int)k + (UP ? (a > b ? 1 : 0) : (a < b ? -1 : 0));
    } else {
        c = (int)(UP ? ceilf(t) : floorf(t));
    }
    return min(127, max(-127, c));
}

// Running elementwise maximum and minimum of a lane's E elements, and whether any was NaN or infinite.
// 16-bit pools keep them packed, two elements an operation.
template <typename T, int E> struct Extremes {
    static constexpr bool PACKED = E % 2 == 0 && (std::is_same<T, __half>::value || std::is_same<T, __nv_bfloat16>::value);
    using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    float hi[E], lo[E];
    uint32_t phi[E / 2 + 1], plo[E / 2 + 1], bad[E / 2 + 1];
    float odd;

    __device__ __forceinline__ void start() {
        if constexpr (PACKED) {
            // the type's infinities: above and below every finite value
            constexpr uint32_t inf = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                phi[i] = inf | 0x80008000u;
                plo[i] = inf;
                bad[i] = 0u;
            }
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                hi[i] = -INFINITY;
                lo[i] = INFINITY;
            }
            odd = 0.f;
        }
    }
    __device__ __forceinline__ void add(const uint32_t* w) {  // packed
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            const Pair x = *reinterpret_cast<const Pair*>(&w[i]);
            Pair h = *reinterpret_cast<Pair*>(&phi[i]), l = *reinterpret_cast<Pair*>(&plo[i]);
            Pair z = *reinterpret_cast<Pair*>(&bad[i]);
            const uint32_t zero = 0u;
            h = __hmax2(h, x);
            l = __hmin2(l, x);
            z = __hfma2(x, *reinterpret_cast<const Pair*>(&zero), z);  // NaN from NaN and infinities
            phi[i] = *reinterpret_cast<uint32_t*>(&h);
            plo[i] = *reinterpret_cast<uint32_t*>(&l);
            bad[i] = *reinterpret_cast<uint32_t*>(&z);
        }
    }
    __device__ __forceinline__ void add(const float* f) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            hi[i] = fmaxf(hi[i], f[i]);
            lo[i] = fminf(lo[i], f[i]);
            odd = fmaf(f[i], 0.f, odd);
        }
    }
    __device__ __forceinline__ void add_careful(const float* f) {  // NaN as 0, infinities as the largest
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float x = isnan(f[i]) ? 0.f : fminf(fmaxf(f[i], -kLargest), kLargest);
            hi[i] = fmaxf(hi[i], x);
            lo[i] = fminf(lo[i], x);
        }
    }
    __device__ __forceinline__ bool is_odd() const {
        if constexpr (PACKED) {
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < E / 2; ++i) any |= bad[i];
            return (any & 0x7fff7fffu) != 0u;
        } else {
            return !(odd == 0.f);
        }
    }
    __device__ __forceinline__ void finish() {
        if constexpr (PACKED) {
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                Elem<T>::unpack(phi[i], hi + 2 * i);
                Elem<T>::unpack(plo[i], lo + 2 * i);
            }
        }
    }
};

// One warp per (request, touched block, kv head): reads the block's rows [0, written) and writes
// its record.  Bound by the rows it reads.
template <typename T, int D>
__global__ void __launch_bounds__(256) block_bounds_kernel(
    unsigned char* __restrict__ bounds, const unsigned char* __restrict__ keys, const int64_t* __restrict__ tables,
    const int64_t* __restrict__ starts, const int64_t* __restrict__ lens, int64_t requests, int64_t width,
    int64_t num_blocks, int block_size, int kv_heads, int64_t most_blocks) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr bool INT4 = std::is_same<T, Int4Tag>::value;
    constexpr int E = bounds_elems<T>(D), N = D / (32 * E);
    using X = Extremes<T, E>;
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
    const int64_t units = requests * most_blocks * kv_heads;
    const int64_t page_bytes = int4_page_bytes(block_size, D);
    for (int64_t u = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += warps) {
        const int64_t rb = (units >> 31) ? u / kv_heads : (int64_t)((uint32_t)u / (uint32_t)kv_heads);
        const int h = (int)(u - rb * kv_heads);
        const int64_t r = (units >> 31) ? rb / most_blocks : (int64_t)((uint32_t)rb / (uint32_t)most_blocks);
        const int64_t start = starts[r], len = lens[r];
        if (start < 0 || len > width * block_size || start >= len) continue;
        const int64_t j = (uint32_t)start / (uint32_t)block_size + (rb - r * most_blocks);
        if (j * block_size >= len) continue;
        const int64_t page = tables[r * width + j];
        if (page < 0 || page >= num_blocks) continue;
        const int rows = (int)min((int64_t)block_size, len - j * block_size);
        X x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i].start();
        const unsigned char* page4 = keys + (page * kv_heads + h) * page_bytes;
        const T* page16 = reinterpret_cast<const T*>(keys) + (page * block_size * kv_heads + h) * (INT4 ? 0 : (int64_t)D);
        auto values4 = [&](int t, int i, float* f) {  // of row t of a 4-bit page
            const float2 sb = __half22float2(
                *reinterpret_cast<const __half2*>(page4 + (int64_t)block_size * (D / 2) + t * 4));
            const float s = fmaxf(sb.x, kInt4StepMin);
            const int d = (i * 32 + lane) * E;
            const unsigned char* src = page4 + (int64_t)t * (D / 2) + d / 2;
            uint32_t word;
            if constexpr (E == 8) word = *reinterpret_cast<const uint32_t*>(src);
            else if constexpr (E == 4) word = *reinterpret_cast<const uint16_t*>(src);
            else if constexpr (E == 2) word = *src;
            else word = *src >> (4 * (d & 1));
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = __fadd_rn(sb.y, __fmul_rn(s, (float)((word >> (4 * e)) & 15u)));
        };
        auto values = [&](int t, int i, float* f) {
            if constexpr (INT4) values4(t, i, f);
            else RowElems<T, E>::load(page16 + (int64_t)t * kv_heads * D, (i * 32 + lane) * E, f);
        };
#pragma unroll 8
        for (int t = 0; t < rows; ++t) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (X::PACKED) {
                    uint32_t w[E / 2];
                    const unsigned char* src =
                        reinterpret_cast<const unsigned char*>(page16 + (int64_t)t * kv_heads * D + (i * 32 + lane) * E);
                    if constexpr (E == 8) {
                        const uint4 v = ld_global_nc(src);
                        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
                    } else if constexpr (E == 4) {
                        const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
                        w[0] = v.x; w[1] = v.y;
                    } else {
                        w[0] = __ldg(reinterpret_cast<const uint32_t*>(src));
                    }
                    x[i].add(w);
                } else {
                    float f[E];
                    values(t, i, f);
                    x[i].add(f);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (x[i].is_odd()) {  // some key is NaN or infinite: again, with care
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    x[i].hi[e] = -kLargest;
                    x[i].lo[e] = kLargest;
                }
                for (int t = 0; t < rows; ++t) {
                    float f[E];
                    values(t, i, f);
                    x[i].add_careful(f);
                }
            } else {
                x[i].finish();
            }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) top = fmaxf(top, fmaxf(fabsf(x[i].hi[e]), fabsf(x[i].lo[e])));
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
        const bool none = top < kBoundsNone;
        const float inv = none ? 0.f : __fdiv_rn(127.f, top);
        unsigned char* rec = bounds + (page * kv_heads + h) * (int64_t)(2 * D + kBoundsPad);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = (i * 32 + lane) * E;
            unsigned char up[E], down[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                up[e] = (unsigned char)(none ? 0 : bound_code<true>(x[i].hi[e], top, inv));
                down[e] = (unsigned char)(none ? 0 : bound_code<false>(x[i].lo[e], top, inv));
            }
            memcpy(__builtin_assume_aligned(rec + d, E), up, E);
            memcpy(__builtin_assume_aligned(rec + D + d, E), down, E);
        }
        if (lane == 0)
            *reinterpret_cast<uint4*>(rec + 2 * D) =
                make_uint4(none ? 0u : __float_as_uint(__fdiv_rn(top, 127.f)), 0u, 0u, 0u);
    }
}

// Values of the bounds of listed blocks: lower and upper [n, kv_heads, D] (zeros for a block outside
// the pool).  A thread takes four dims of a record.
static __global__ void __launch_bounds__(256) read_bounds_kernel(
    const unsigned char* __restrict__ bounds, const int64_t* __restrict__ ids, int64_t n, int64_t num_blocks,
    int kv_heads, int D, FastDiv quads_of, FastDiv heads_of, float* __restrict__ lower, float* __restrict__ upper) {
    griddep_wait();
    griddep_launch_dependents();
    const int64_t rows = n * kv_heads;
    // rows in pieces of 2^20, so that a piece's quads are counted in 31 bits
    for (int64_t r0 = 0; r0 < rows; r0 += 1 << 20) {
        const uint32_t quads = (uint32_t)min(rows - r0, (int64_t)(1 << 20)) * quads_of.d;
#pragma unroll 2
        for (uint32_t u = blockIdx.x * blockDim.x + threadIdx.x; u < quads; u += gridDim.x * blockDim.x) {
            const uint32_t in = quads_of(u);
            const int d = (int)(u - in * quads_of.d) * 4;
            const int64_t row = r0 + in;
            const int64_t at = (rows >> 31) ? row / kv_heads : (int64_t)heads_of((uint32_t)row);
            const int64_t id = ids[at];
            float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
            if (id >= 0 && id < num_blocks) {
                const unsigned char* rec = bounds + (id * kv_heads + (row - at * kv_heads)) * (int64_t)(2 * D + kBoundsPad);
                const float s = *reinterpret_cast<const float*>(rec + 2 * D);
                const char4 a = *reinterpret_cast<const char4*>(rec + d), b = *reinterpret_cast<const char4*>(rec + D + d);
                hi = make_float4(a.x * s, a.y * s, a.z * s, a.w * s);
                lo = make_float4(b.x * s, b.y * s, b.z * s, b.w * s);
            }
            *reinterpret_cast<float4*>(lower + row * D + d) = lo;
            *reinterpret_cast<float4*>(upper + row * D + d) = hi;
        }
    }
}

// ------------------------------------------------------------------ scores
// Keys that order as their scores do: 0 for a block that cannot be selected (no page of the pool),
// the largest for one that has to be, else a whole number that grows with the score.
__device__ __forceinline__ uint32_t score_key(float score) {
    const uint32_t b = __float_as_uint(score + 0.f);  // -0 counts as +0
    const uint32_t k = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return min(0xfffffffeu, max(1u, k));
}

constexpr int kScoreHeads = 8;   // kv heads a CTA scores
constexpr int kScoreSpan = 512;  // blocks a CTA scores at most

struct SelectParams {
    const void* q;
    const unsigned char* bounds;
    const int64_t* tables;
    const int64_t* lens;
    uint32_t* keys;     // [batch, kv_heads, width]
    int64_t* selected;  // [batch, kv_heads, take]
    int64_t width, num_blocks;
    int q_heads, kv_heads, group, block_size, take, sink, recent;
    int span;  // blocks a CTA scores
};

__device__ __forceinline__ int blocks_of(const SelectParams& p, int64_t b) {
    const int64_t len = p.lens[b];
    return len > 0 && len <= p.width * p.block_size ? (int)((len + p.block_size - 1) / p.block_size) : 0;
}

// Scores of p.span blocks of one request for up to kScoreHeads kv heads.  Bound by the
// records' bytes.  16 bytes of codes a lane: int4_row_lanes(D) lanes a head.  The spans are as long
// as fills the device once (a CTA first makes the query's codes, 3 us), and a span's keys go out
// head by head from shared memory.
template <typename T, int D, bool FULL>  // FULL: eight heads in every group
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) score_blocks_kernel(const SelectParams p) {
    constexpr int LPH = int4_row_lanes(D);        // lanes a head (2 D / 16 of them active)
    constexpr int HPW = 32 / LPH;                 // heads a warp scores at once
    constexpr int PASSES = kScoreHeads / HPW;
    constexpr int REC = 2 * D + kBoundsPad;
    __shared__ float sums[kScoreHeads][2 * D];
    __shared__ int tops[kScoreHeads];
    __shared__ __align__(16) signed char codes[kScoreHeads][2 * D];
    __shared__ uint32_t found[kScoreHeads][kScoreSpan];
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t chunks = (p.width + p.span - 1) / p.span;
    const int64_t b = blockIdx.x / chunks;
    const int n = blocks_of(p, b);
    const int first = (int)(blockIdx.x - b * chunks) * p.span;
    if (first >= n || n <= p.take) return;  // a request with no more blocks than are taken needs no scores
    const int h0 = blockIdx.y * kScoreHeads, nh = min(kScoreHeads, p.kv_heads - h0);
    // ---- blocks: warp w takes blocks w, w + 8, ... of the span, AHEAD at a time, the next ones loaded
    // while these are scored (the first while the query's codes are made); lane x looks up the page of
    // the warp's next x-th block for 32 of them at once
    constexpr int AHEAD = 2;
    const int sub = lane % LPH, part = lane / LPH;
    const bool active = sub * 16 < 2 * D;
    const int last = min(n, first + p.span), mine = (last - first - warp + 7) / 8;
    const int64_t* table = p.tables + b * p.width + first + warp;
    const int recent_from = n - p.recent;
    const int64_t stride = p.kv_heads * (int64_t)REC;
    const unsigned char* lane_at = p.bounds + (int64_t)(h0 + part) * REC + (active ? sub * 16 : 0);
    // The sums of the passes are halved across the lanes of a head as they are added up, so that a lane
    // ends with the sum of one pass: head my_head, complete in the lanes that are `out`.
    int my_pass = 0;
#pragma unroll
    for (int half = PASSES / 2, m = LPH / 2; half > 0; half /= 2, m /= 2) my_pass += (lane & m) ? half : 0;
    const int my_head = my_pass * HPW + part;
    const bool out = sub % (LPH / PASSES) == 0 && my_head < nh;
    const unsigned char* scale_at = p.bounds + (int64_t)(h0 + min(my_head, nh - 1)) * REC + 2 * D;
    struct Records {
        int4 v[AHEAD][PASSES];
        float scale[AHEAD];
        bool ok[AHEAD];
    };
    int64_t page = 0;
    auto load = [&](Records& r, int k0) {
        if (k0 % 32 == 0) {
            const int k = k0 + lane;
            page = k < mine ? table[8 * k] : -1;
            if (page >= p.num_blocks) page = -1;
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int64_t id = __shfl_sync(0xffffffffu, page, (k0 + a) % 32);
            r.ok[a] = id >= 0;
            const int64_t off = (r.ok[a] ? id : 0) * stride;
            const unsigned char* rec = lane_at + off;
            r.scale[a] = __ldg(reinterpret_cast<const float*>(scale_at + off));
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                // a group of fewer heads reads its first again
                const unsigned char* at = rec + (FULL || i * HPW + part < nh ? i * HPW * REC : -part * REC);
                const uint4 w = ld_global_nc(at);
                r.v[a][i] = make_int4((int)w.x, (int)w.y, (int)w.z, (int)w.w);
            }
        }
    };
    Records even, odd;
    load(even, 0);
    // ---- the query's codes
    if (tid < kScoreHeads) tops[tid] = 0;
    __syncthreads();
    const T* q = static_cast<const T*>(p.q) + (b * p.q_heads + (int64_t)h0 * p.group) * D;
    for (int x = tid; x < nh * D; x += 256) {
        const int h = x / D, d = x - h * D;
        float pos = 0.f, neg = 0.f;
        for (int i = 0; i < p.group; ++i) {
            const float f = Elem<T>::to_float(q[(int64_t)(h * p.group + i) * D + d]);
            const float v = isnan(f) ? 0.f : fminf(fmaxf(f, -kLargest), kLargest);
            pos += fmaxf(v, 0.f);
            neg += fminf(v, 0.f);
        }
        pos = fminf(pos, kLargest);
        neg = fmaxf(neg, -kLargest);
        sums[h][d] = pos;
        sums[h][D + d] = neg;
        // non-negative floats order as their bits; a warp's 32 dims are of one head, and all of its lanes
        // are here (nh * D is a multiple of 32)
        const int top = __reduce_max_sync(0xffffffffu, __float_as_int(fmaxf(pos, -neg)));
        if (lane == 0) atomicMax(&tops[h], top);
    }
    __syncthreads();
    for (int x = tid; x < kScoreHeads * 2 * D; x += 256) {
        const int h = x / (2 * D), d = x - h * (2 * D);
        float c = 0.f;
        if (h < nh) {
            const float top = __int_as_float(tops[h]);
            c = top < kBoundsNone ? 0.f : rintf(__fmul_rn(sums[h][d], __fdiv_rn(127.f, top)));
        }
        codes[h][d] = (signed char)min(127, max(-127, (int)c));
    }
    __syncthreads();
    int4 qc[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
        qc[i] = active ? *reinterpret_cast<const int4*>(&codes[i * HPW + part][sub * 16]) : make_int4(0, 0, 0, 0);
    auto score = [&](const Records& r, int k0) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            int dot[PASSES];
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                dot[i] = __dp4a(r.v[a][i].x, qc[i].x, 0);
                dot[i] = __dp4a(r.v[a][i].y, qc[i].y, dot[i]);
                dot[i] = __dp4a(r.v[a][i].z, qc[i].z, dot[i]);
                dot[i] = __dp4a(r.v[a][i].w, qc[i].w, dot[i]);
            }
#pragma unroll
            for (int half = PASSES / 2, m = LPH / 2; m > 0; half /= 2, m /= 2) {
                const bool upper = lane & m;
#pragma unroll
                for (int i = 0; i < (half > 0 ? half : 1); ++i) {
                    const int keep = half > 0 && upper ? dot[i + half] : dot[i];
                    const int give = half > 0 && !upper ? dot[i + half] : dot[i];
                    dot[i] = keep + __shfl_xor_sync(0xffffffffu, give, m);
                }
            }
            if (out && k0 + a < mine) {
                const int j = first + warp + 8 * (k0 + a);
                const float s = __fmul_rn((float)dot[0], r.scale[a]);
                uint32_t key = isnan(s) ? 1u : score_key(s);
                if (j < p.sink || j >= recent_from) key = 0xffffffffu;
                found[my_head][j - first] = r.ok[a] ? key : 0u;
            }
        }
    };
#pragma unroll 1
    for (int k0 = 0; k0 < mine; k0 += 2 * AHEAD) {
        if (k0 + AHEAD < mine) load(odd, k0 + AHEAD);
        score(even, k0);
        if (k0 + 2 * AHEAD < mine) load(even, k0 + 2 * AHEAD);
        if (k0 + AHEAD < mine) score(odd, k0 + AHEAD);
    }
    __syncthreads();
    for (int h = 0; h < nh; ++h)
        for (int x = tid; x < last - first; x += 256)
            p.keys[(b * p.kv_heads + h0 + h) * p.width + first + x] = found[h][x];
}

// ------------------------------------------------------------------ selection
// One CTA per (request, kv head): the `take` largest keys, ties to the lowest
// block, in the order of the blocks.  The take-th largest key is found eight
// bits at a time from a histogram; a block scan of the counts gives every
// selected block its place.  Keys are held in shared memory when they fit.
constexpr int kSelectThreads = 512;
constexpr int kSelectHeld = 24576;  // keys in shared memory (96 KB)

// Sums of x and y over the CTA, in one barrier: `turn` alternates between two sets of warp sums.
__device__ __forceinline__ uint2 block_sum2(uint32_t x, uint32_t y, uint2 (*sums)[32], int turn) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    x = __reduce_add_sync(0xffffffffu, x);
    y = __reduce_add_sync(0xffffffffu, y);
    if (lane == 0) sums[turn & 1][threadIdx.x >> 5] = make_uint2(x, y);
    __syncthreads();
    const uint2 s = lane < warps ? sums[turn & 1][lane] : make_uint2(0u, 0u);
    return make_uint2(__reduce_add_sync(0xffffffffu, s.x), __reduce_add_sync(0xffffffffu, s.y));
}

// Requests of up to 4096 blocks: a thread holds KEYS consecutive keys in registers, and the
// take-th largest is found two bits at a time, three counts and a barrier each, until a value is met
// that exactly `take` keys reach (a score's 32 bits rarely tie).
template <int KEYS>
__global__ void __launch_bounds__(512) select_few_kernel(const SelectParams p) {
    __shared__ int counts[2][32];
    __shared__ uint2 sums[2][32];
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int64_t b = blockIdx.x / p.kv_heads;
    const int n = blocks_of(p, b);
    int64_t* out = p.selected + (int64_t)blockIdx.x * p.take;
    const bool all = n <= p.take;
    uint32_t key[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
        const int at = tid * KEYS + i;
        key[i] = 0;
        if (at < n) {
            if (all) {
                const int64_t page = p.tables[b * p.width + at];
                key[i] = page >= 0 && page < p.num_blocks ? 0xffffffffu : 0u;
            } else {
                key[i] = __ldcg(p.keys + (int64_t)blockIdx.x * p.width + at);
            }
        }
    }
    // the largest value that `take` keys reach: 0 where fewer have a page
    uint32_t threshold = 0;
    int above = 0;  // keys over it
    int turn = 0;
    if (!all) {
        const uint32_t take = (uint32_t)p.take;
        for (int shift = 30; shift >= 0; shift -= 2) {
            const uint32_t one = threshold | (1u << shift), two = threshold | (2u << shift), three = threshold | (3u << shift);
            uint32_t c12 = 0, c3 = 0;  // counts of two probes share a word: a CTA has 4096 keys at most
#pragma unroll
            for (int i = 0; i < KEYS; ++i) {
                c12 += (key[i] >= one ? 1u : 0u) + (key[i] >= two ? 65536u : 0u);
                c3 += key[i] >= three;
            }
            const uint2 s = block_sum2(c12, c3, sums, turn++);
            const uint32_t n1 = s.x & 0xffffu, n2 = s.x >> 16, n3 = s.y;
            const uint32_t reached = n3 >= take ? n3 : n2 >= take ? n2 : n1;
            threshold = n3 >= take ? three : n2 >= take ? two : n1 >= take ? one : threshold;
            if (reached == take) break;  // exactly the keys from here on
        }
        uint32_t count = 0;
#pragma unroll
        for (int i = 0; i < KEYS; ++i) count += key[i] > threshold;
        above = (int)block_sum2(count, 0u, sums, turn++).x;
    }
    __syncthreads();
    const int ties = all ? 0 : p.take - above;
    // places, in the order of the blocks
    int more = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
        more += key[i] > threshold;
        equal += key[i] == threshold && key[i] != 0;
    }
    int im = more, ie = equal;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int vm = __shfl_up_sync(0xffffffffu, im, off), ve = __shfl_up_sync(0xffffffffu, ie, off);
        if (lane >= off) {
            im += vm;
            ie += ve;
        }
    }
    if (lane == 31) {
        counts[0][warp] = im;
        counts[1][warp] = ie;
    }
    __syncthreads();
    int wm = lane < warps ? counts[0][lane] : 0, we = lane < warps ? counts[1][lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int vm = __shfl_up_sync(0xffffffffu, wm, off), ve = __shfl_up_sync(0xffffffffu, we, off);
        if (lane >= off) {
            wm += vm;
            we += ve;
        }
    }
    const int all_more = __shfl_sync(0xffffffffu, wm, 31), all_equal = __shfl_sync(0xffffffffu, we, 31);
    const int before_m = __shfl_sync(0xffffffffu, wm, max(0, warp - 1)), before_e = __shfl_sync(0xffffffffu, we, max(0, warp - 1));
    more = im - more + (warp ? before_m : 0);
    equal = ie - equal + (warp ? before_e : 0);
    int place = more + min(equal, ties);
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
        const bool tie = key[i] == threshold && key[i] != 0;
        if (key[i] > threshold || (tie && equal < ties)) out[place++] = tid * KEYS + i;
        equal += tie;
    }
    for (int i = all_more + min(all_equal, ties) + tid; i < p.take; i += blockDim.x) out[i] = -1;
}

// Exclusive prefix over the block of (a, b); total in *ta, *tb.
__device__ __forceinline__ void block_prefix2(int& a, int& b, int* ta, int* tb, int (*scratch)[kSelectThreads / 32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int ia = a, ib = b;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int va = __shfl_up_sync(0xffffffffu, ia, off), vb = __shfl_up_sync(0xffffffffu, ib, off);
        if (lane >= off) {
            ia += va;
            ib += vb;
        }
    }
    __syncthreads();
    if (lane == 31) {
        scratch[0][warp] = ia;
        scratch[1][warp] = ib;
    }
    __syncthreads();
    int sa = 0, sb = 0, wa = 0, wb = 0;
#pragma unroll
    for (int w = 0; w < kSelectThreads / 32; ++w) {
        if (w == warp) {
            wa = sa;
            wb = sb;
        }
        sa += scratch[0][w];
        sb += scratch[1][w];
    }
    a = wa + ia - a;
    b = wb + ib - b;
    *ta = sa;
    *tb = sb;
}

static __global__ void __launch_bounds__(kSelectThreads) select_blocks_kernel(const SelectParams p, int held_max) {
    extern __shared__ uint32_t held[];
    __shared__ int hist[256];
    __shared__ int scratch[2][kSelectThreads / 32];
    __shared__ uint32_t found_digit;
    __shared__ int found_above;
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x;
    const int64_t b = blockIdx.x / p.kv_heads;
    const int n = blocks_of(p, b);
    int64_t* out = p.selected + (int64_t)blockIdx.x * p.take;
    const uint32_t* keys = p.keys + (int64_t)blockIdx.x * p.width;
    const int64_t* table = p.tables + b * p.width;
    const bool all = n <= p.take;  // every block that has a page
    const bool held_on = n <= held_max;
    auto key_at = [&](int i) -> uint32_t {
        if (held_on) return held[i];
        if (all) {
            const int64_t page = table[i];
            return page >= 0 && page < p.num_blocks ? 0xffffffffu : 0u;
        }
        return keys[i];
    };
    if (held_on) {
        for (int i = tid; i < n; i += kSelectThreads) {
            if (all) {
                const int64_t page = table[i];
                held[i] = page >= 0 && page < p.num_blocks ? 0xffffffffu : 0u;
            } else {
                held[i] = __ldcg(keys + i);
            }
        }
    }
    __syncthreads();
    // ---- the take-th largest key: `prefix` its leading digits, `above` how many keys exceed them
    uint32_t threshold = 0;
    int ties = 0;  // how many keys equal to the threshold are taken
    if (!all) {
        uint32_t prefix = 0;
        int above = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i0 = 0; i0 < n; i0 += kSelectThreads) {
                const int i = i0 + tid;
                const uint32_t k = i < n ? key_at(i) : 0u;
                const bool in = i < n && (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)));
                const uint32_t digit = (k >> shift) & 255u;
                // one atomic for a warp whose keys share the digit (the first digit nearly always)
                const unsigned live = __ballot_sync(0xffffffffu, in);
                if (live) {
                    const int lead = __ffs(live) - 1;
                    const uint32_t d0 = __shfl_sync(0xffffffffu, digit, lead);
                    if (__all_sync(0xffffffffu, !in || digit == d0)) {
                        if ((tid & 31) == lead) atomicAdd(&hist[d0], __popc(live));
                    } else if (in) {
                        atomicAdd(&hist[digit], 1);
                    }
                }
            }
            __syncthreads();
            if (tid < 32) {  // the digit at which the count from the top reaches `take`
                int c[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    c[i] = hist[255 - (tid * 8 + i)];
                    sum += c[i];
                }
                int incl = sum;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, incl, off);
                    if (tid >= off) incl += v;
                }
                int run = above + incl - sum;
                if (run < p.take && run + sum >= p.take) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (run < p.take && run + c[i] >= p.take) {
                            found_digit = 255 - (tid * 8 + i);
                            found_above = run;
                        }
                        run += c[i];
                    }
                }
            }
            __syncthreads();
            prefix |= found_digit << shift;
            above = found_above;
        }
        threshold = prefix;
        ties = p.take - above;
    }
    // ---- places, in the order of the blocks: each thread counts a run of them.  Keys above the
    // threshold are taken, and the first `ties` equal to it (never a block without a page).
    const int per = (n + kSelectThreads - 1) / kSelectThreads;
    const int lo = min(n, tid * per), hi = min(n, lo + per);
    int more = 0, equal = 0, all_more, all_equal;
    for (int i = lo; i < hi; ++i) {
        const uint32_t k = key_at(i);
        more += k > threshold;
        equal += k == threshold && k != 0;
    }
    block_prefix2(more, equal, &all_more, &all_equal, scratch);
    int place = more + min(equal, ties), seen = equal;
    for (int i = lo; i < hi; ++i) {
        const uint32_t k = key_at(i);
        const bool tie = k == threshold && k != 0;
        if (k > threshold || (tie && seen < ties)) out[place++] = i;
        seen += tie;
    }
    const int count = all_more + min(all_equal, ties);
    for (int i = count + tid; i < p.take; i += kSelectThreads) out[i] = -1;
}

}  // namespace minikv
