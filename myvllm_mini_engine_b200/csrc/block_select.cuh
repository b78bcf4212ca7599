// Selecting the blocks a query attends: key bounds of every block, and the
// blocks of highest score.
//
// Bounds.  [num_blocks, kv_heads, 2 D + 16] bytes: D int8 codes of the keys'
// elementwise maximum over the block's rows, D of their minimum, one fp32 scale
// (12 bytes of padding).  scale = top / 127 with top the largest magnitude of
// the 2 D bounds; codes ceil(127 max / top) and floor(127 min / top), so that
// code * scale bounds the keys.  A block whose top is below 2^-100 has zero
// codes and scale.  NaN keys count as 0, infinite ones as the largest fp32.
//
// Score.  For a kv head with query heads q_1 .. q_n, let qp = sum_h max(q_h, 0)
// and qn = sum_h min(q_h, 0) (fp32, in the order of the heads).  Then for any
// key k of the block, sum_h q_h . k <= sum_d max_d qp_d + min_d qn_d.  The 2 D
// values (qp, qn) are held in 8 bits over their largest magnitude, a factor
// common to all blocks of the kv head, so
//   score = scale_block * (sum_d maxcode_d qpcode_d + mincode_d qncode_d)
// where the sum is a whole number below 2^24: it has one value whatever the
// order, and with it the selection.  8-bit bounds are a sixteenth of the bytes
// of a 16-bit block of 16 tokens (K and V: 64 D bytes).
#pragma once

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
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
    const int64_t units = requests * most_blocks * kv_heads;
    const int64_t page_bytes = int4_page_bytes(block_size, D);
    for (int64_t u = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += warps) {
        const int64_t rb = u / kv_heads;
        const int h = (int)(u - rb * kv_heads);
        const int64_t r = rb / most_blocks;
        const int64_t start = starts[r], len = lens[r];
        if (start < 0 || len > width * block_size) continue;
        const int64_t j = start / block_size + (rb - r * most_blocks);
        if (start >= len || j * block_size >= len) continue;
        const int64_t page = tables[r * width + j];
        if (page < 0 || page >= num_blocks) continue;
        const int rows = (int)min((int64_t)block_size, len - j * block_size);
        float hi[N][E], lo[N][E];
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                hi[i][e] = -kLargest;
                lo[i][e] = kLargest;
            }
        const unsigned char* page4 = keys + (page * kv_heads + h) * page_bytes;
#pragma unroll 4
        for (int t = 0; t < rows; ++t) {
            float f[N][E];
            if constexpr (INT4) {
                const float2 sb = __half22float2(
                    *reinterpret_cast<const __half2*>(page4 + (int64_t)block_size * (D / 2) + t * 4));
                const float s = fmaxf(sb.x, kInt4StepMin);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int d = (i * 32 + lane) * E;
                    const unsigned char* src = page4 + (int64_t)t * (D / 2) + d / 2;
                    uint32_t word;
                    if constexpr (E == 8) word = *reinterpret_cast<const uint32_t*>(src);
                    else if constexpr (E == 4) word = *reinterpret_cast<const uint16_t*>(src);
                    else if constexpr (E == 2) word = *src;
                    else word = *src >> (4 * (d & 1));
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        f[i][e] = __fadd_rn(sb.y, __fmul_rn(s, (float)((word >> (4 * e)) & 15u)));
                }
            } else {
                const T* row = reinterpret_cast<const T*>(keys) +
                               ((page * block_size + t) * kv_heads + h) * (int64_t)D;
#pragma unroll
                for (int i = 0; i < N; ++i) RowElems<T, E>::load(row, (i * 32 + lane) * E, f[i]);
            }
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = isnan(f[i][e]) ? 0.f : fminf(fmaxf(f[i][e], -kLargest), kLargest);
                    hi[i][e] = fmaxf(hi[i][e], x);
                    lo[i][e] = fminf(lo[i][e], x);
                }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) top = fmaxf(top, fmaxf(fabsf(hi[i][e]), fabsf(lo[i][e])));
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
        const bool none = top < kBoundsNone;
        const float inv = none ? 0.f : __fdiv_rn(127.f, top);
        unsigned char* rec = bounds + (page * kv_heads + h) * (int64_t)(2 * D + kBoundsPad);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = (i * 32 + lane) * E;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                rec[d + e] = (unsigned char)(none ? 0 : bound_code<true>(hi[i][e], top, inv));
                rec[D + d + e] = (unsigned char)(none ? 0 : bound_code<false>(lo[i][e], top, inv));
            }
        }
        if (lane == 0)
            *reinterpret_cast<uint4*>(rec + 2 * D) =
                make_uint4(none ? 0u : __float_as_uint(__fdiv_rn(top, 127.f)), 0u, 0u, 0u);
    }
}

// Values of the bounds of listed blocks: lower and upper [n, kv_heads, D] (zeros for a block outside the pool).
static __global__ void __launch_bounds__(256) read_bounds_kernel(
    const unsigned char* __restrict__ bounds, const int64_t* __restrict__ ids, int64_t n, int64_t num_blocks,
    int kv_heads, int D, float* __restrict__ lower, float* __restrict__ upper) {
    griddep_wait();
    griddep_launch_dependents();
    const int64_t quads = n * kv_heads * (D / 4);
    for (int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; u < quads; u += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = u / (D / 4);
        const int d = (int)(u - row * (D / 4)) * 4;
        const int64_t id = ids[row / kv_heads];
        float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
        if (id >= 0 && id < num_blocks) {
            const unsigned char* rec = bounds + (id * kv_heads + row % kv_heads) * (int64_t)(2 * D + kBoundsPad);
            const float s = *reinterpret_cast<const float*>(rec + 2 * D);
            const char4 a = *reinterpret_cast<const char4*>(rec + d), b = *reinterpret_cast<const char4*>(rec + D + d);
            hi = make_float4(a.x * s, a.y * s, a.z * s, a.w * s);
            lo = make_float4(b.x * s, b.y * s, b.z * s, b.w * s);
        }
        *reinterpret_cast<float4*>(lower + row * D + d) = lo;
        *reinterpret_cast<float4*>(upper + row * D + d) = hi;
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

constexpr int kScoreHeads = 8;    // kv heads a CTA scores
constexpr int kScoreBlocks = 64;  // blocks a CTA scores

struct SelectParams {
    const void* q;
    const unsigned char* bounds;
    const int64_t* tables;
    const int64_t* lens;
    uint32_t* keys;     // [batch, kv_heads, width]
    int64_t* selected;  // [batch, kv_heads, take]
    int64_t width, num_blocks;
    int q_heads, kv_heads, group, block_size, take, sink, recent;
};

__device__ __forceinline__ int blocks_of(const SelectParams& p, int64_t b) {
    const int64_t len = p.lens[b];
    return len > 0 && len <= p.width * p.block_size ? (int)((len + p.block_size - 1) / p.block_size) : 0;
}

// Scores of kScoreBlocks blocks of one request for up to kScoreHeads kv heads.  Bound by the
// records' bytes.  16 bytes of codes a lane: int4_row_lanes(D) lanes a head.
template <typename T, int D>
__global__ void __launch_bounds__(256) score_blocks_kernel(const SelectParams p) {
    constexpr int LPH = int4_row_lanes(D);        // lanes a head (2 D / 16 of them active)
    constexpr int HPW = 32 / LPH;                 // heads a warp scores at once
    constexpr int PASSES = kScoreHeads / HPW > 0 ? kScoreHeads / HPW : 1;
    constexpr int REC = 2 * D + kBoundsPad;
    __shared__ float sums[kScoreHeads][2 * D];
    __shared__ int tops[kScoreHeads];
    __shared__ __align__(16) signed char codes[kScoreHeads][2 * D];
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t chunks = (p.width + kScoreBlocks - 1) / kScoreBlocks;
    const int64_t b = blockIdx.x / chunks;
    const int n = blocks_of(p, b);
    const int first = (int)(blockIdx.x - b * chunks) * kScoreBlocks;
    if (first >= n || n <= p.take) return;  // a request with no more blocks than are taken needs no scores
    const int h0 = blockIdx.y * kScoreHeads, nh = min(kScoreHeads, p.kv_heads - h0);
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
        atomicMax(&tops[h], __float_as_int(fmaxf(pos, -neg)));  // non-negative floats order as their bits
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
    const int sub = lane % LPH, part = lane / LPH;
    const bool active = sub * 16 < 2 * D;
    int4 qc[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
        qc[i] = active ? *reinterpret_cast<const int4*>(&codes[i * HPW + part][sub * 16]) : make_int4(0, 0, 0, 0);
    // ---- blocks: 8 warps, one block each at a time
    const int last = min(n, first + kScoreBlocks);
    const int64_t* table = p.tables + b * p.width;
    const int recent_from = n - p.recent;
#pragma unroll 2
    for (int j = first + warp; j < last; j += 8) {
        const int64_t page = table[j];
        const bool ok = page >= 0 && page < p.num_blocks;
        const unsigned char* rec = p.bounds + ((ok ? page : 0) * p.kv_heads + h0) * (int64_t)REC;
        int4 v[PASSES];
        float scale[PASSES];
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int h = min(i * HPW + part, nh - 1);
            v[i] = make_int4(0, 0, 0, 0);
            if (active) {
                const uint4 w = ld_global_nc(rec + (int64_t)h * REC + sub * 16);
                v[i] = make_int4((int)w.x, (int)w.y, (int)w.z, (int)w.w);
            }
            scale[i] = *reinterpret_cast<const float*>(rec + (int64_t)h * REC + 2 * D);
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            int dot = __dp4a(v[i].x, qc[i].x, 0);
            dot = __dp4a(v[i].y, qc[i].y, dot);
            dot = __dp4a(v[i].z, qc[i].z, dot);
            dot = __dp4a(v[i].w, qc[i].w, dot);
#pragma unroll
            for (int m = LPH / 2; m > 0; m >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, m);
            const int h = i * HPW + part;
            if (sub == 0 && h < nh) {
                const float s = __fmul_rn((float)dot, scale[i]);
                uint32_t key = isnan(s) ? 1u : score_key(s);
                if (j < p.sink || j >= recent_from) key = 0xffffffffu;
                p.keys[(b * p.kv_heads + h0 + h) * p.width + j] = ok ? key : 0u;
            }
        }
    }
}

// ------------------------------------------------------------------ selection
// One CTA per (request, kv head): the `take` largest keys, ties to the lowest
// block, in the order of the blocks.  The take-th largest key is found eight
// bits at a time from a histogram; a block scan of the counts gives every
// selected block its place.  Keys are held in shared memory when they fit.
constexpr int kSelectThreads = 512;
constexpr int kSelectHeld = 24576;  // keys in shared memory (96 KB)

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
