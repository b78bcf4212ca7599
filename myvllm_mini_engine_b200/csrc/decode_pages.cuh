// Decode attention over lists of pages: a 4-bit pool (every page of a request,
// or selected ones) and selected pages of a 16-bit pool.
//
//   s_t = q . k_t / sqrt(D),   out = sum_t softmax(s)_t v_t
//
// over the tokens t of the listed pages.  For the 4-bit pool k_t = base_t +
// step_t c_t and v_t = base'_t + step'_t c'_t (int4_pool.cuh), so
//   s_t = (step_t (q . c_t) + base_t sum(q)) / sqrt(D)
//   out = (sum_t P'_t c'_t + sum_t P_t base'_t) / sum_t P_t,   P'_t = P_t step'_t
// and the codes enter the matrix products exactly, with no arithmetic of their
// own: a nibble left in the low bits of a half is the fp16 subnormal c 2^-24
// (c 2^-20 for the high nibbles), so a mask makes an operand register and the
// powers of two are taken out of the fp32 results.  The running maximum is that
// of log2 P' = s + log2(step'), so that P' fits fp16 whatever the steps are; P =
// P' / step' stays in fp32.
//
// Split.  A unit is (request, kv head, up to 8 of its query heads).  The tiles
// (TT tokens) of all units form one list, cut into equal runs, one per CTA of a
// grid that fills the device once, so ragged lengths cost no balance and a
// captured graph stays valid when lengths change.  In a CTA the warps take the
// tiles of its run in turn.  Each warp has its own ring of stages, filled by
// its own 16-byte asynchronous copies: no producer warp and no barrier until a
// unit's tiles end, where the warps' states are joined through shared memory in
// a fixed order.  A unit that spans CTAs leaves one partial per CTA; the CTA
// that takes the unit's last ticket joins them, in the order of the CTAs.
//
// Long batches are bound by the instructions that make the operands: 636 a
// tile of 32 tokens at D = 128, where the SM could issue 760 in the time that its
// share of the memory's rate brings the tile, and the 16 warps that the registers
// allow keep it at half of that (256 requests of 4096 tokens, 8 kv heads: 235 us,
// 4.9 TB/s of the pool, against 177 us at the measured copy rate; 275 in a run of
// seconds, when the power limit takes the clock to 1650 MHz).  Small ones are
// bound by the chain of launch, look-ups, pages and join (8 x 513: 13 us).
// Copies a lane rather than bulk copies of a slice (1 KB of codes at D = 128):
// those took a tenth longer, with more instructions, for the barriers.  mma.sync rather
// than tcgen05: the group's few query heads are the N = 8 columns, and the
// operands are made in registers.
#pragma once

#include "common.cuh"
#include "int4_pool.cuh"

namespace minikv {

struct PageDecodeParams {
    const void* q;
    const unsigned char* kc;
    const unsigned char* vc;
    const int64_t* tables;
    const int64_t* lens;
    const int64_t* selected;  // [batch, kv_heads, take] logical blocks, or null: all
    void* out;
    float* partial;           // [units + runs][heads][D]
    float* lse;               // [units + runs][heads], log2
    unsigned int* tickets;    // [units], zero before and after
    int batch, q_heads, kv_heads, group, chunks, heads;  // heads: query heads of a unit's record, min(group, 8)
    int num_blocks, block_size, width, take;
    uint64_t bs_magic;        // v / block_size = v * bs_magic >> 42 for v < 2^20
    int64_t page_stride;      // bytes of a page (all kv heads)
    int64_t head_stride;      // bytes from one kv head's part of a page to the next
    int64_t row_stride;       // bytes from one token's row to the next
    float scale_log2;         // log2(e) / sqrt(D)
};

// ------------------------------------------------------------ PTX wrappers
// 16 (or 4) bytes global -> shared; the bytes past `bytes` are zeros and are not read.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// 8x8 matrix of 16-bit elements, transposed across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float log2_fast(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t permute_bytes(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a b, with nothing added
__device__ __forceinline__ void mma16816_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// max over the 8 lanes that share a column of an accumulator (lanes of equal lane % 4)
__device__ __forceinline__ float column_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}
__device__ __forceinline__ float column_sum(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 4);
    x += __shfl_xor_sync(0xffffffffu, x, 8);
    return x + __shfl_xor_sync(0xffffffffu, x, 16);
}

// m, which the exponents are taken against, lies kHeadroom below the running maximum (log2), so that P
// uses fp16's range (65504) and not only its part below 1: a token keeps all bits of P down to 2^-26 of
// the largest, and is lost below 2^-37 of it, so that a million tokens lose 2^-17 of the weight at most
// (with the maximum at 1, 2^-25 and 2^-5).  m is raised only when a score exceeds the maximum that it was
// made for by more than 2^3: P <= 2^15, O is rescaled once or twice a unit, and the maximum over a
// column's lanes is taken only then: a vote tells.
constexpr float kHeadroom = 12.f, kMost = 15.f;

// The fp16 query of a 4-bit pool is scaled by a power of two so that a row's largest element lies in
// [2^14, 2^15): elements keep all of their bits down to 2^-24 of the largest (odd ones, stored 16 times
// smaller, too), and below that are off by 2^-35 of it at most.
constexpr int kQueryTop = 14;
// The exponent of the largest element less kQueryTop, kept where 2^-e and 2^e are both normal.
__device__ __forceinline__ int query_exponent(float top) {
    const int e = (int)((__float_as_uint(top) >> 23) & 255) - 127 - kQueryTop;
    return top > 0.f && top < INFINITY ? min(120, max(-120, e)) : 0;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

constexpr uint32_t kNibbleMask = 0x000f000fu;  // the low nibbles of two halves
constexpr float kCodeScale = 16777216.f;       // 2^24: a nibble in the low bits of a half is code 2^-24

// ---------------------------------------------------------------- consumers
// Both keep, per warp: m (kHeadroom below the running maximum, log2), l (lane's part of sum P),
// z (4-bit: lane's part of sum P base'), o (accumulators) of the unit's query
// heads; lane (g, q4) = (lane / 4, lane % 4) holds columns (heads) 2 q4, 2 q4 + 1.

// 4-bit pool, 32 tokens a tile in two slices of 16 (the M rows of K Q^T; one
// maximum and one rescale for both).  Row r < 8 of a slice's MMA is its token
// r / 2 + 4 (r % 2) (+ 8 for r >= 8): a lane's V loads of one instruction then
// are of four neighbouring tokens.  The order of the head dims in a dot product
// is free: lane q4 takes dims q4 D/4 .. of K (whole words of codes) and, for
// V^T (dims are the M rows), lane g dims g D/8 ..: in each four of them nibble
// 0 and 2 are rows g and g + 8 of one MMA; another takes the whole bytes, n0 +
// 16 n1 and n2 + 16 n3 (a byte in the low bits of a half is still a subnormal),
// and the odd nibbles' sums are the difference at the end: a fifth fewer
// integer operations than masking both.  For K the odd nibbles are masked out
// in place (16 times larger as subnormals) and meet a Q scaled by 1/16.
// A lane first turns the (step, base) pairs of one token into what the scores
// and the sums need, for the whole warp: done by every lane for its own rows it
// took a sixth of the tile's instructions.
// P' goes in as two fp16 terms (2^-22): one (2^-12) would move a twentieth of a
// bf16 output's roundings to the next value.  TWIN: a unit of up to four heads
// holds them twice, in columns 0..3 and again in 4..7, so the same scores and P' come
// out there; those columns multiply the second term, and their sums are added at
// the unit's end: no MMA more than one term takes (256 x 4096 tokens, D = 128,
// two heads a kv head, in a long run: one term 269 us, this 278, a second set of
// MMAs 293).  O of a tile is summed by itself and added to the unit's: 234.8 us
// against 233.7 with MMAs that add to the unit's, at eight heads a kv head 275
// against 258 (registers spill).
template <typename T, int D, bool TWIN>
struct Int4Consumer {
    static constexpr int TT = 32;
    static constexpr int RB = D / 2;                         // bytes of a row's codes
    static constexpr int kRowBytes = RB;                     // ... staged without padding
    static constexpr int kPairs = TT * 2 * RB;               // stage: K codes, V codes, K pairs, V pairs
    static constexpr int kStageBytes = kPairs + TT * 8;
    static constexpr int kScratch = TT * 20;                 // per warp: the tokens' factors
    static constexpr int NW = D / 32;                        // words of K a lane takes of a row
    static constexpr int NH = D / 32;                        // 16-bit runs of V a lane takes of a row
    static constexpr int kPieces = NH;                       // groups of 32 output dims

    uint32_t qb[2 * NW][2];
    float o[2 * NH][4];
    float m[2], l[2], z[2], qsum[2], qscale[2];
    int g, q4, lane;

    __device__ void setup(int lane_) {
        lane = lane_;
        g = lane >> 2;
        q4 = lane & 3;
    }

    // Q of head g in fp16, scaled (kQueryTop)
    __device__ void begin(const T* q, int heads, float scale_log2) {
        float f[8 * NW];
        float top = 0.f;
        const int head = TWIN ? g & 3 : g;
        if (head < heads) {
#pragma unroll
            for (int i = 0; i < 8 * NW; i += 8) {
                Elem<T>::load(*reinterpret_cast<const uint4*>(q + head * D + q4 * (D / 4) + i), f + i);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[i + e]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8 * NW; ++i) f[i] = 0.f;
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = query_exponent(top);
        const float down = power_of_two(-e);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float unit = (i & 1) ? 0.0625f : 1.f;
                x[i] = __half2float(__float2half_rn(f[8 * w + i] * down * unit));
                sum += (i & 1) ? x[i] * 16.f : x[i];
            }
            qb[2 * w][0] = Elem<__half>::pack(x[0], x[4]);
            qb[2 * w][1] = Elem<__half>::pack(x[2], x[6]);
            qb[2 * w + 1][0] = Elem<__half>::pack(x[1], x[5]);
            qb[2 * w + 1][1] = Elem<__half>::pack(x[3], x[7]);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const float up = power_of_two(e) * scale_log2;
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // of the heads this lane's accumulators hold
            qsum[h] = __shfl_sync(0xffffffffu, sum, (2 * q4 + h) * 4);
            qscale[h] = __shfl_sync(0xffffffffu, up, (2 * q4 + h) * 4);
            m[h] = -INFINITY;
            l[h] = z[h] = 0.f;
        }
#pragma unroll
        for (int t = 0; t < 2 * NH; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][i] = 0.f;
    }

    // K words of one row for this lane
    __device__ __forceinline__ void load_k(const unsigned char* p, uint32_t* w) const {
        if constexpr (NW % 4 == 0) {
#pragma unroll
            for (int i = 0; i < NW / 4; ++i) {
                const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * i);
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
        } else if constexpr (NW % 2 == 0) {
#pragma unroll
            for (int i = 0; i < NW / 2; ++i) {
                const uint2 v = *reinterpret_cast<const uint2*>(p + 8 * i);
                w[2 * i] = v.x; w[2 * i + 1] = v.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NW; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
        }
    }
    // V: 16-bit runs i of the rows of two tokens, side by side (the first token's in the low half)
    __device__ __forceinline__ void load_v(const unsigned char* a, const unsigned char* b, uint32_t* x) const {
        if constexpr (NH % 2 == 0) {
            uint32_t wa[NH / 2], wb[NH / 2];
            if constexpr (NH % 8 == 0) {
                const uint4 u = *reinterpret_cast<const uint4*>(a), v = *reinterpret_cast<const uint4*>(b);
                wa[0] = u.x; wa[1] = u.y; wa[2] = u.z; wa[3] = u.w;
                wb[0] = v.x; wb[1] = v.y; wb[2] = v.z; wb[3] = v.w;
            } else if constexpr (NH % 4 == 0) {
                const uint2 u = *reinterpret_cast<const uint2*>(a), v = *reinterpret_cast<const uint2*>(b);
                wa[0] = u.x; wa[1] = u.y;
                wb[0] = v.x; wb[1] = v.y;
            } else {
#pragma unroll
                for (int i = 0; i < NH / 2; ++i) {
                    wa[i] = *reinterpret_cast<const uint32_t*>(a + 4 * i);
                    wb[i] = *reinterpret_cast<const uint32_t*>(b + 4 * i);
                }
            }
#pragma unroll
            for (int i = 0; i < NH / 2; ++i) {
                x[2 * i] = permute_bytes(wa[i], wb[i], 0x5410u);
                x[2 * i + 1] = permute_bytes(wa[i], wb[i], 0x7632u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NH; ++i)
                x[i] = *reinterpret_cast<const uint16_t*>(a + 2 * i) |
                       ((uint32_t) * reinterpret_cast<const uint16_t*>(b + 2 * i) << 16);
        }
    }

    // Raise the maxima to those of the columns, where they exceed them by the slack.
    __device__ __forceinline__ void raise(const float* top) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float mx = column_max(top[h]);
            if (mx > m[h] + kMost) {
                const float alpha = exp2_fast(m[h] - (mx - kHeadroom));
                m[h] = mx - kHeadroom;
                l[h] *= alpha;
                z[h] *= alpha;
#pragma unroll
                for (int x = 0; x < 2 * NH; ++x) {
                    o[x][h] *= alpha;
                    o[x][h + 2] *= alpha;
                }
            }
        }
    }

    __device__ __forceinline__ void tile(const unsigned char* stage, uint32_t valid, float, unsigned char* scratch) {
        const unsigned char* kst = stage;
        const unsigned char* vst = stage + TT * RB;
        float4* factors = reinterpret_cast<float4*>(scratch);        // [TT]: K step 2^24, K base, log2 V step, 1 / V step
        float* weights = reinterpret_cast<float*>(scratch + TT * 16);  // [TT]: V base / V step
        {
            const __half2* pairs = reinterpret_cast<const __half2*>(stage + kPairs);
            const float2 k = __half22float2(pairs[lane]), v = __half22float2(pairs[TT + lane]);
            const float vs = fmaxf(v.x, kInt4StepMin);
            const float inv = rcp_fast(vs);
            // a masked token (its codes and pairs are zeros) drops out by log2 P' = -inf
            factors[lane] = make_float4(fmaxf(k.x, kInt4StepMin) * kCodeScale, k.y,
                                        (valid >> lane) & 1u ? log2_fast(vs) : -INFINITY, inv);
            weights[lane] = v.y * inv;
        }
        __syncwarp();
        const int row = (g >> 1) + 4 * (g & 1);
        float t[2][4], rinv[2][2], rbase[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r0 = 16 * i + row, r1 = r0 + 8;
            uint32_t k0[NW], k1[NW];
            load_k(kst + r0 * RB + q4 * (RB / 4), k0);
            load_k(kst + r1 * RB + q4 * (RB / 4), k1);
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const uint32_t a[4] = {k0[w] & kNibbleMask, k1[w] & kNibbleMask, (k0[w] >> 8) & kNibbleMask,
                                       (k1[w] >> 8) & kNibbleMask};
                mma16816<__half>(s, a, qb[2 * w][0], qb[2 * w][1]);
                const uint32_t b[4] = {k0[w] & (kNibbleMask << 4), k1[w] & (kNibbleMask << 4),
                                       (k0[w] >> 8) & (kNibbleMask << 4), (k1[w] >> 8) & (kNibbleMask << 4)};
                mma16816<__half>(s, b, qb[2 * w + 1][0], qb[2 * w + 1][1]);
            }
            const float4 f0 = factors[r0], f1 = factors[r1];
            rinv[i][0] = f0.w;
            rinv[i][1] = f1.w;
            rbase[i][0] = weights[r0];
            rbase[i][1] = weights[r1];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                t[i][h] = fmaf(fmaf(s[h], f0.x, f0.y * qsum[h]), qscale[h], f0.z);
                t[i][h + 2] = fmaf(fmaf(s[h + 2], f1.x, f1.y * qsum[h]), qscale[h], f1.z);
            }
        }
        float top[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) top[h] = fmaxf(fmaxf(t[0][h], t[0][h + 2]), fmaxf(t[1][h], t[1][h + 2]));
        if (__any_sync(0xffffffffu, top[0] > m[0] + kMost || top[1] > m[1] + kMost)) raise(top);
        const float mm[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};  // 2^(-inf - 0) = 0
        uint32_t w[2][2], w2[2][2];  // P' of a slice, transposed: the terms that this lane's columns multiply
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = exp2_fast(t[i][e] - mm[e & 1]);
                l[e & 1] = fmaf(p[e], rinv[i][e >> 1], l[e & 1]);
                z[e & 1] = fmaf(p[e], rbase[i][e >> 1], z[e & 1]);
            }
            const uint32_t p01 = Elem<__half>::pack(p[0], p[1]), p23 = Elem<__half>::pack(p[2], p[3]);
            float back[4];
            Elem<__half>::unpack(p01, back);
            Elem<__half>::unpack(p23, back + 2);
            const uint32_t r01 = Elem<__half>::pack(p[0] - back[0], p[1] - back[1]);
            const uint32_t r23 = Elem<__half>::pack(p[2] - back[2], p[3] - back[3]);
            const bool second = TWIN && q4 >= 2;
            w[i][0] = transpose8x8(second ? r01 : p01);
            w[i][1] = transpose8x8(second ? r23 : p23);
            if constexpr (!TWIN) {
                w2[i][0] = transpose8x8(r01);
                w2[i][1] = transpose8x8(r23);
            }
        }
        uint32_t x[2][2][NH];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const unsigned char* v = vst + (16 * i + q4) * RB + g * (RB / 8);
            load_v(v, v + 4 * RB, x[i][0]);
            load_v(v + 8 * RB, v + 12 * RB, x[i][1]);
        }
        // O of the tile by itself, then added: an MMA truncates its sum, which the codes (none negative)
        // would turn into a bias that grows with the tokens
#pragma unroll
        for (int u = 0; u < NH; ++u) {
            float even[4], whole[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t b[4] = {x[i][0][u] & 0x00ff00ffu, permute_bytes(x[i][0][u], 0u, 0x4341u),
                                       x[i][1][u] & 0x00ff00ffu, permute_bytes(x[i][1][u], 0u, 0x4341u)};
                const uint32_t a[4] = {b[0] & kNibbleMask, b[1] & kNibbleMask, b[2] & kNibbleMask, b[3] & kNibbleMask};
                if (i == 0) {
                    mma16816_first(even, a, w[i][0], w[i][1]);
                    mma16816_first(whole, b, w[i][0], w[i][1]);
                } else {
                    mma16816<__half>(even, a, w[i][0], w[i][1]);
                    mma16816<__half>(whole, b, w[i][0], w[i][1]);
                }
                if constexpr (!TWIN) {
                    mma16816<__half>(even, a, w2[i][0], w2[i][1]);
                    mma16816<__half>(whole, b, w2[i][0], w2[i][1]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[2 * u][e] += even[e];
                o[2 * u + 1][e] += whole[e];
            }
        }
    }

    // A unit's end: the second terms' sums join the first ones'.
    __device__ __forceinline__ void finish() {
        if constexpr (TWIN) {
#pragma unroll
            for (int x = 0; x < 2 * NH; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[x][i] += __shfl_xor_sync(0xffffffffu, o[x][i], 2);
        }
    }

    // Piece u of the accumulators times f[h]: element [head % 4][x] for x < 32 is output dim dim_of(u, x).
    __device__ __forceinline__ void put_piece(int u, const float* f, float* dst) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float k = f[h] * kCodeScale;
            *reinterpret_cast<float4*>(dst + ((2 * q4 + h) & 3) * 32 + 4 * g) =
                make_float4(o[2 * u][h] * k, high(u, h) * k, o[2 * u][h + 2] * k, high(u, h + 2) * k);
        }
    }
    // sums of the odd nibbles, from those of the even ones and of the bytes
    __device__ __forceinline__ float high(int u, int i) const { return (o[2 * u + 1][i] - o[2 * u][i]) * 0.0625f; }
    __device__ static __forceinline__ int dim_of(int u, int x) { return (x >> 2) * (D / 8) + 4 * u + (x & 3); }
    // The lane's part of head 2 q4 + h: (O + add) * inv into a row of V (fp32 or T).
    template <typename V> __device__ __forceinline__ void put_row(int h, float add, float inv, V* row) const {
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            const float f[4] = {fmaf(o[2 * u][h], kCodeScale, add) * inv, fmaf(high(u, h), kCodeScale, add) * inv,
                                fmaf(o[2 * u][h + 2], kCodeScale, add) * inv,
                                fmaf(high(u, h + 2), kCodeScale, add) * inv};
            V* dst = row + g * (D / 8) + 4 * u;
            if constexpr (sizeof(V) == 4) *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
            else *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<V>::pack(f[0], f[1]), Elem<V>::pack(f[2], f[3]));
        }
    }
};

// 16-bit pool, 16 tokens a tile; K and V rows are padded by 16 bytes so that
// the 8 rows of an ldmatrix meet different banks.  P goes in as two terms of the
// pool's type, as in the decode over whole tables.
template <typename T, int D>
struct Wide16Consumer {
    static constexpr int TT = 16;
    static constexpr int RB = 2 * D;
    static constexpr int kRowBytes = RB + 16;
    static constexpr int kPairs = 0;
    static constexpr int kStageBytes = TT * 2 * kRowBytes;
    static constexpr int kScratch = 0;
    static constexpr int KSTEPS = D / 16;
    static constexpr int kPieces = D / 32;

    uint32_t qb[KSTEPS][2];
    float o[KSTEPS][4];
    float m[2], l[2], z[2];
    int g, q4, k_off, v_off;

    __device__ void setup(int lane) {
        g = lane >> 2;
        q4 = lane & 3;
        const int r = lane & 7, mat = lane >> 3;
        k_off = (r + 8 * (mat & 1)) * kRowBytes + 16 * (mat >> 1);
        v_off = TT * kRowBytes + (r + 8 * (mat >> 1)) * kRowBytes + 16 * (mat & 1);
    }

    __device__ void begin(const T* q, int heads, float) {
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
            const T* p = q + g * D + 16 * k + 2 * q4;
            qb[k][0] = g < heads ? *reinterpret_cast<const uint32_t*>(p) : 0u;
            qb[k][1] = g < heads ? *reinterpret_cast<const uint32_t*>(p + 8) : 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[k][i] = 0.f;
        }
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = z[0] = z[1] = 0.f;
    }

    __device__ __forceinline__ void raise(const float* top) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float mx = column_max(top[h]);
            if (mx > m[h] + kMost) {
                const float alpha = exp2_fast(m[h] - (mx - kHeadroom));
                m[h] = mx - kHeadroom;
                l[h] *= alpha;
#pragma unroll
                for (int x = 0; x < KSTEPS; ++x) {
                    o[x][h] *= alpha;
                    o[x][h + 2] *= alpha;
                }
            }
        }
    }

    __device__ __forceinline__ void tile(const unsigned char* stage, uint32_t valid, float scale_log2, unsigned char*) {
        const uint32_t base = smem_addr(stage);
        float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
            uint32_t a[4];
            ldmatrix4(base + k_off + 32 * k, a);
            mma16816<T>((k & 1) ? s2 : s, a, qb[k][0], qb[k][1]);
        }
        const bool ok0 = (valid >> g) & 1u, ok1 = (valid >> (g + 8)) & 1u;
        s[0] = ok0 ? (s[0] + s2[0]) * scale_log2 : -INFINITY;
        s[1] = ok0 ? (s[1] + s2[1]) * scale_log2 : -INFINITY;
        s[2] = ok1 ? (s[2] + s2[2]) * scale_log2 : -INFINITY;
        s[3] = ok1 ? (s[3] + s2[3]) * scale_log2 : -INFINITY;
        const float top[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
        if (__any_sync(0xffffffffu, top[0] > m[0] + kMost || top[1] > m[1] + kMost)) raise(top);
        const float mm[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};  // 2^(-inf - 0) = 0
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[e] = exp2_fast(s[e] - mm[e & 1]);
            l[e & 1] += p[e];
        }
        const uint32_t p01 = Elem<T>::pack(p[0], p[1]), p23 = Elem<T>::pack(p[2], p[3]);
        float back[4];
        Elem<T>::unpack(p01, back);
        Elem<T>::unpack(p23, back + 2);
        const uint32_t b0 = transpose8x8(p01), b1 = transpose8x8(p23);
        const uint32_t c0 = transpose8x8(Elem<T>::pack(p[0] - back[0], p[1] - back[1]));
        const uint32_t c1 = transpose8x8(Elem<T>::pack(p[2] - back[2], p[3] - back[3]));
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
            uint32_t a[4];
            ldmatrix4_trans(base + v_off + 32 * k, a);
            mma16816<T>(o[k], a, c0, c1);
            mma16816<T>(o[k], a, b0, b1);
        }
    }

    __device__ __forceinline__ void finish() {}

    __device__ __forceinline__ void put_piece(int u, const float* f, float* dst) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* row = dst + ((2 * q4 + h) & 3) * 32 + g;
            row[0] = o[2 * u][h] * f[h];
            row[8] = o[2 * u][h + 2] * f[h];
            row[16] = o[2 * u + 1][h] * f[h];
            row[24] = o[2 * u + 1][h + 2] * f[h];
        }
    }
    __device__ static __forceinline__ int dim_of(int u, int x) { return 32 * u + x; }
    template <typename V> __device__ __forceinline__ void put_row(int h, float add, float inv, V* row) const {
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
            row[16 * k + g] = Elem<V>::from_float((o[k][h] + add) * inv);
            row[16 * k + g + 8] = Elem<V>::from_float((o[k][h + 2] + add) * inv);
        }
    }
};

// ------------------------------------------------------------------ the kernel
template <typename Consumer, bool INT4> struct PageShape {
    static constexpr int kWarps = INT4 ? 8 : 4;
    static constexpr int kStages = 3;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kStage = Consumer::kStageBytes + 16;  // and the mask of its tokens
    static constexpr int kPiece = kWarps * 4 * 32 * 4;         // one piece of every warp's accumulators, four heads
    static constexpr int kWork = kWarps * Consumer::kScratch > kPiece ? kWarps * Consumer::kScratch : kPiece;
    // rings | consumers' scratch, or a piece | warps' (m, l, z) of 8 heads | slices | prefix of tiles
    static constexpr int kScratch = kWarps * kStages * kStage;
    static constexpr int kStats = kScratch + kWork;
    static constexpr int kSlices = kStats + kWarps * 8 * 3 * 4;
    static constexpr int kPrefix = kSlices + kWarps * 16 * 16;
    static constexpr int kBytes = kPrefix + (kThreads + 4) * 4;
};

// A place in the list of tiles: tile j of unit ul of request b, whose units have `tiles` tiles each
// and whose list has `len` tokens.
struct TileCursor {
    int b, ul, j, tiles, len;
};

// 16 tokens of one page: where their codes (rows) start in the pool, their (step, base) pairs
// relative to that, and which of them exist.
struct __align__(16) PageSlice {
    int64_t at;
    int pairs;
    uint32_t mask;
};

// Warps of a 4-bit pool's decode work alone where each gets this many tiles, and a unit is as long as this
// many of their runs at most (so it has up to two partials more).
constexpr int kLeastAlone = 5, kMostPartials = 8;

// Joins n partials of a unit, in their order, into its output rows: `threads` threads share the
// heads x D elements, four each at a time.  Up to four partials are loaded at once.
template <typename T, int D>
__device__ void join_partials(const PageDecodeParams& p, int64_t first, int n, int heads, int64_t qh0, int thread,
                              int threads) {
    constexpr int AT_ONCE = 4;
#pragma unroll 2
    for (int x = thread; x < heads * (D / 4); x += threads) {
        const int head = x / (D / 4), d = (x - head * (D / 4)) * 4;
        const float* lse = p.lse + first * p.heads + head;
        const float4* part = reinterpret_cast<const float4*>(p.partial + (first * p.heads + head) * D + d);
        float mx = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < n; k0 += AT_ONCE) {
            float e[AT_ONCE];
            float4 v[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int64_t at = min(k0 + k, n - 1);
                e[k] = __ldcg(lse + at * p.heads);
                v[k] = __ldcg(part + at * p.heads * (D / 4));
                if (k0 + k >= n) e[k] = -INFINITY;
            }
            float top = mx;
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) top = fmaxf(top, e[k]);
            const float keep = mx == -INFINITY ? 0.f : exp2_fast(mx - top);
            sum *= keep;
            acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const float w = e[k] == -INFINITY ? 0.f : exp2_fast(e[k] - top);
                sum += w;
                acc = make_float4(fmaf(w, v[k].x, acc.x), fmaf(w, v[k].y, acc.y), fmaf(w, v[k].z, acc.z),
                                  fmaf(w, v[k].w, acc.w));
            }
            mx = top;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (qh0 + head) * D + d) =
            make_uint2(Elem<T>::pack(acc.x * inv, acc.y * inv), Elem<T>::pack(acc.z * inv, acc.w * inv));
    }
}

// ALIGNED: block_size is a multiple of 16, so that a slice of 16 tokens lies in one page.
template <typename T, int D, typename Consumer, bool INT4, bool SELECTED, bool ALIGNED>
__global__ void __launch_bounds__(PageShape<Consumer, INT4>::kThreads, D <= 128 ? 2 : 1)
    page_decode_kernel(const PageDecodeParams p) {
    using Shape = PageShape<Consumer, INT4>;
    constexpr int TT = Consumer::TT, W = Shape::kWarps, NS = Shape::kStages, RB = Consumer::RB, STAGE = Shape::kStage;
    extern __shared__ __align__(128) unsigned char smem[];
    float* piece = reinterpret_cast<float*>(smem + Shape::kScratch);
    float* stats = reinterpret_cast<float*>(smem + Shape::kStats);  // [3][W][8]
    int* prefix = reinterpret_cast<int*>(smem + Shape::kPrefix);    // [threads + 1]: tiles before a thread's requests
    __shared__ int warp_sums[W], warp_most[W];
    __shared__ int last_ticket;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int B = p.batch, U = p.kv_heads * p.chunks;
    const int64_t cap = (int64_t)p.width * p.block_size;

    griddep_wait();
    griddep_launch_dependents();

    // Tokens of a request's list: its length, or the rows of its listed blocks (a block past the
    // request's last or a -1 is masked token by token).
    auto usable = [&](int b) -> int {
        const int64_t len = p.lens[b];
        return len > 0 && len <= cap ? (int)len : 0;
    };
    auto tiles_of = [&](int len) -> int {
        if (SELECTED) {
            const int blocks = min(p.take, (len + p.block_size - 1) / p.block_size);
            return (blocks * p.block_size + TT - 1) / TT;
        }
        return (len + TT - 1) / TT;
    };
    // ---- exclusive prefix of the tile counts: a thread has `per` requests (one, for a batch of up to
    // W * 32), and those within a thread's are counted again where needed, so any batch fits
    const int per = (B + W * 32 - 1) / (W * 32);
    {
        const int lo = min(B, tid * per), hi = min(B, lo + per);
        int sum = 0, most = 0;
        for (int i = lo; i < hi; ++i) {
            const int n = tiles_of(usable(i));
            sum += n;
            most = max(most, n);
            if (n == 0 && i % gridDim.x == blockIdx.x)  // nothing to attend: zeros
                for (int x = 0; x < p.q_heads * D; x += 8)
                    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)i * p.q_heads * D + x) =
                        make_uint4(0u, 0u, 0u, 0u);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) warp_most[warp] = most;
        int incl = sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += v;
        }
        if (lane == 31) warp_sums[warp] = incl;
        __syncthreads();
        int run = incl - sum;
        for (int w = 0; w < warp; ++w) run += warp_sums[w];
        prefix[tid] = run;
        if (tid == W * 32 - 1) prefix[W * 32] = run + sum;
        __syncthreads();
    }
    // ---- teams and their runs of tiles.  A team is the CTA, whose warps take the tiles of its run in
    // turn and join at the end of each unit, or a single warp with a run of its own: no barrier, an
    // eighth of the joins, but a unit is then cut into as many partials as warps share it.  The figures
    // come from the lengths, so all CTAs agree.  A CTA and a warp, D = 128, 8 kv heads: 256 x 4096 tokens
    // (111 tiles a warp, a unit of 1.2 runs) 274 and 235 us, 64 x 4096 (28, 5) 82 and 73, 64 lists of 1024
    // (7, 5) 37 and 31, 32 x 4096 (14, 9) 48 and 46, 32 lists of 2048 (7, 9) 33 and 31, 12 x 4096 (5, 25) 27
    // and 29, 32 x 1024 (3.5, 9) 17 and 22, 1 x 131072 (14, 296) 46 and 102.  A 16-bit pool's four warps are
    // faster together: 64 lists of 2048 tokens 99 and 101 us, 32 of them 57 and 61.
    const int64_t total = (int64_t)prefix[W * 32] * U;
    int longest = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) longest = max(longest, warp_most[w]);
    const int64_t slots = (int64_t)gridDim.x * W;
    const bool alone = INT4 && total >= kLeastAlone * slots && longest * slots <= kMostPartials * total;
    const int TW = alone ? 1 : W, rank = alone ? 0 : warp;  // warps of the team, and this one's place
    const int64_t team = alone ? (int64_t)blockIdx.x * W + warp : blockIdx.x;
    int64_t G = (int64_t)gridDim.x * (alone ? W : 1);  // runs
    // Every run has a tile, of a CTA at least one for each warp; where that is no more than four a warp,
    // a whole unit's, which then needs no join (8 x 513 tokens: 17.8 -> 11.6 us when it was introduced).
    const int least = longest <= 4 * W ? max(W, longest) : W;
    G = min(G, alone ? total : (total + least - 1) / least);
    if (team >= G) return;
    const int64_t t0 = team * total / G;
    const int run = (int)((team + 1) * total / G - t0);  // the team's tiles; its warp r takes tiles r, r + TW, ...

    const int searched = (B - 1) / per;  // the last thread that has requests
    auto cursor_at = [&](int64_t t) -> TileCursor {
        const int64_t x = t / U;  // tiles of the requests before (and of the own one's units, divided)
        int lo = 0, hi = searched;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] <= x) lo = mid; else hi = mid - 1;
        }
        TileCursor c;
        c.b = lo * per;
        int64_t before = prefix[lo];
        for (;; ++c.b) {
            c.len = usable(c.b);
            c.tiles = tiles_of(c.len);
            if (x < before + c.tiles || c.b == B - 1) break;
            before += c.tiles;
        }
        const int in = (int)(t - before * U);
        c.ul = in / c.tiles;
        c.j = in - c.ul * c.tiles;
        return c;
    };
    auto advance = [&](TileCursor& c, int by) {
        c.j += by;
        while (c.j >= c.tiles) {
            c.j -= c.tiles;
            if (++c.ul == U) {
                c.ul = 0;
                do {
                    if (++c.b >= B) return;
                    c.len = usable(c.b);
                    c.tiles = tiles_of(c.len);
                } while (c.tiles == 0);
            }
        }
    };

    // ---- the warp's copies: tile k of the warp is tile rank + k TW of the run.
    // Aligned: lane x < 16 looks up slice x % SPT of tile x / SPT of a batch of TPB tiles, whose slices lie
    // in shared memory while the next batch is looked up in two steps (listed block, then page), so that
    // no step waits for a load of its own.  Otherwise lane r looks up token r of the next tile.
    unsigned char* ring = smem + warp * NS * STAGE;
    const uint32_t ring_addr = smem_addr(ring);
    const int mine = run > rank ? (run - rank + TW - 1) / TW : 0;
    constexpr int SPT = TT / 16, TPB = 16 / SPT;
    constexpr int CPR = RB / 16;  // 16-byte pieces of a row
    PageSlice* slices = reinterpret_cast<PageSlice*>(smem + Shape::kSlices) + warp * 16;
    const int in_tile = ALIGNED ? (lane % SPT) * 16 : (TT == 32 ? lane : lane & 15);  // this lane's first token of the tile
    int look_k = ALIGNED ? (lane & 15) / SPT : 0;                                     // and its tile, of the warp's
    TileCursor look = {0, 0, 0, 0, 0};
    if (look_k < mine) look = cursor_at(t0 + rank + (int64_t)look_k * TW);
    int64_t block = -1;  // looked up: the listed block
    int page = -1;       // and its page
    auto place = [&](int& e, int& off) {  // of this lane's token in the list: entry and row
        const int v = look.j * TT + in_tile;
        e = (int)(((uint64_t)(uint32_t)v * p.bs_magic) >> 42);
        off = v - e * p.block_size;
    };
    auto kv_head = [&]() { return p.chunks == 1 ? look.ul : look.ul / p.chunks; };
    auto look_block = [&]() {
        block = -1;
        if (look_k < mine) {
            int e, off;
            place(e, off);
            if (SELECTED) {
                if (e < p.take) block = p.selected[((int64_t)look.b * p.kv_heads + kv_head()) * p.take + e];
            } else {
                block = e;
            }
        }
    };
    auto look_page = [&]() {
        page = -1;
        if (block >= 0 && block < p.width) {
            int e, off;
            place(e, off);
            if ((int)block * p.block_size + off < look.len) {
                const int64_t id = p.tables[(int64_t)look.b * p.width + block];
                if (id >= 0 && id < p.num_blocks) page = (int)id;
            }
        }
    };
    auto look_on = [&](int by) {
        look_k += by;
        if (look_k < mine) advance(look, by * TW);
    };
    auto keep_batch = [&]() {
        PageSlice s;
        s.at = 0;
        s.pairs = 0;
        s.mask = 0;
        if (page >= 0) {
            int e, off;
            place(e, off);
            const int left = look.len - ((int)block * p.block_size + off);
            s.mask = left >= 16 ? 0xffffu : (1u << left) - 1u;
            s.at = (int64_t)page * p.page_stride + (int64_t)kv_head() * p.head_stride + off * p.row_stride;
            if (INT4) s.pairs = p.block_size * RB + off * 4 - off * RB;
        }
        __syncwarp();
        if (lane < 16) slices[lane] = s;
        __syncwarp();
    };
    // a whole slice of K or of V is PIECES pieces a lane, when those divide evenly
    constexpr bool EVEN = CPR % 2 == 0 && (INT4 || 32 % CPR == 0);
    constexpr int PIECES = CPR / 2, CPR_ = 32 % CPR == 0 ? CPR : 32;
    const int64_t lane_from = INT4 ? lane * 16 : (int64_t)(lane / CPR_) * p.row_stride + lane % CPR_ * 16;
    const uint32_t lane_to = ring_addr + (INT4 ? lane * 16 : lane / CPR_ * Consumer::kRowBytes + lane % CPR_ * 16);
    const unsigned char* k_lane = p.kc + lane_from;
    const int64_t v_from_k = (int64_t)(reinterpret_cast<uintptr_t>(p.vc) - reinterpret_cast<uintptr_t>(p.kc));
    int copied = 0;          // tiles copied
    uint32_t copy_at = 0;    // stage of the next one, as an offset in the ring
    auto copy_aligned = [&]() {
        const int i = copied % TPB;
        if (i == 0 && copied) keep_batch();
        if (i == 0) {
            look_on(TPB);
            look_block();
        }
        if (i == TPB / 2) look_page();
        uint32_t valid = 0;
#pragma unroll
        for (int s = 0; s < SPT; ++s) {
            const PageSlice sl = slices[i * SPT + s];
            valid |= sl.mask << (16 * s);
            const unsigned char* ks = k_lane + sl.at;
            const unsigned char* vs = ks + v_from_k;
            const uint32_t to = lane_to + copy_at + 16 * s * Consumer::kRowBytes;
            if (EVEN && sl.mask == 0xffffu) {  // the usual slice: whole
#pragma unroll
                for (int x = 0; x < PIECES; ++x) {
                    const int64_t step = INT4 ? x * 512 : x * (32 / CPR_) * p.row_stride;
                    const uint32_t at = to + (INT4 ? x * 512 : x * (32 / CPR_) * Consumer::kRowBytes);
                    copy16(at, ks + step, 16u);
                    copy16(at + TT * Consumer::kRowBytes, vs + step, 16u);
                }
            } else {  // 16 CPR pieces of K, then as many of V
#pragma unroll 1
                for (int x = 0; x < CPR; ++x) {
                    const int c = x * 32 + lane;
                    const bool is_v = c >= 16 * CPR;
                    const int in = is_v ? c - 16 * CPR : c;
                    const int row = in / CPR;
                    const bool on = (sl.mask >> row) & 1u;
                    const int64_t from = on ? (int64_t)row * p.row_stride + (in - row * CPR) * 16 : 0;
                    copy16(ring_addr + copy_at + ((is_v ? TT : 0) + 16 * s + row) * Consumer::kRowBytes + (in - row * CPR) * 16,
                           (is_v ? p.vc : p.kc) + sl.at + from, on ? 16u : 0u);
                }
            }
        }
        if (INT4 && lane < 8 * SPT) {  // pairs: 64 bytes of K and of V a slice
            const PageSlice sl = slices[i * SPT + (lane >> 3)];
            const int x = lane & 3, have = __popc(sl.mask) * 4 - x * 16, left = min(16, max(0, have));
            const unsigned char* src = p.kc + ((lane & 4) ? v_from_k : 0) + sl.at + sl.pairs + (left ? x * 16 : 0);
            copy16(ring_addr + copy_at + Consumer::kPairs + ((lane & 4) ? TT * 4 : 0) + (lane >> 3) * 64 + x * 16, src,
                   (uint32_t)left);
        }
        if (lane == 0) *reinterpret_cast<uint32_t*>(ring + copy_at + Consumer::kStageBytes) = valid;
    };
    auto copy_rows = [&]() {
        const uint32_t dst = ring_addr + copy_at;
        int e, page_off;
        place(e, page_off);
        const uint32_t valid = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) *reinterpret_cast<uint32_t*>(ring + copy_at + Consumer::kStageBytes) = valid;
        const int64_t head = (int64_t)kv_head() * p.head_stride;
#pragma unroll
        for (int c0 = 0; c0 < TT * CPR; c0 += 32) {
            const int c = c0 + lane;
            const int r = min(c / CPR, TT - 1), x = c - (c / CPR) * CPR;
            const int pg = __shfl_sync(0xffffffffu, page, r), off = __shfl_sync(0xffffffffu, page_off, r);
            if (TT * CPR % 32 == 0 || c < TT * CPR) {
                const int64_t at = pg < 0 ? 0 : pg * p.page_stride + head + off * p.row_stride + x * 16;
                const uint32_t n = pg < 0 ? 0u : 16u;
                copy16(dst + r * Consumer::kRowBytes + x * 16, p.kc + at, n);
                copy16(dst + (TT + r) * Consumer::kRowBytes + x * 16, p.vc + at, n);
            }
        }
        if (INT4) {
            const int64_t at = page < 0 ? 0 : page * p.page_stride + head + (int64_t)p.block_size * RB + page_off * 4;
            copy4(dst + Consumer::kPairs + lane * 4, p.kc + at, page < 0 ? 0u : 4u);
            copy4(dst + Consumer::kPairs + TT * 4 + lane * 4, p.vc + at, page < 0 ? 0u : 4u);
        }
        look_on(1);
        look_block();
        look_page();
    };
    auto copy_tile = [&]() {
        if (copied < mine) {
            if constexpr (ALIGNED) copy_aligned();
            else copy_rows();
            ++copied;
            copy_at = copy_at == (NS - 1) * STAGE ? 0 : copy_at + STAGE;
        }
        copy_commit();
    };
    look_block();
    look_page();
    if constexpr (ALIGNED) keep_batch();
#pragma unroll 1
    for (int s = 0; s < NS; ++s) copy_tile();
    bool first = true;  // the warp's first tile frees no stage

    Consumer c;
    c.setup(lane);
    unsigned char* scratch = smem + Shape::kScratch + warp * Consumer::kScratch;
    uint32_t stage = 0;
    int t = rank;  // the warp's next tile, of the run
    TileCursor seg = cursor_at(t0);
    for (int done = 0; done < run;) {
        // ---- one unit's tiles in the team's run: [done, end)
        const int end = min(run, done + seg.tiles - seg.j);
        const int kvh = seg.ul / p.chunks, chunk = seg.ul - kvh * p.chunks;
        const int heads = min(8, p.group - 8 * chunk);
        const int64_t qh0 = (int64_t)seg.b * p.q_heads + kvh * p.group + 8 * chunk;
        c.begin(static_cast<const T*>(p.q) + qh0 * D, heads, p.scale_log2);
        for (; t < end; t += TW) {
            if (first) copy_wait<NS - 1>(); else copy_wait<NS - 2>();
            __syncwarp();  // the stage is whole, and the one filled next has been read by every lane
            if (!first) copy_tile();
            first = false;
            c.tile(ring + stage, *reinterpret_cast<const uint32_t*>(ring + stage + Consumer::kStageBytes), p.scale_log2,
                   scratch);
            stage = stage == (NS - 1) * STAGE ? 0 : stage + STAGE;
        }
        c.finish();
        const bool whole = seg.j == 0 && end - done == seg.tiles;
        const int64_t unit = (int64_t)seg.b * U + seg.ul;
        const int64_t record = unit + team;  // grows by at least one from segment to segment
        const int64_t unit_lo = t0 + done - seg.j;
        // runs that hold the unit's first and last tile
        auto owner = [&](int64_t x) { return (int)(((x + 1) * G + total - 1) / total) - 1; };
        if (alone) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float L = column_sum(c.l[h]), Z = column_sum(c.z[h]);
                const int head = 2 * c.q4 + h;
                const float inv = L == 0.f ? 0.f : 1.f / L;
                if (head < heads) {
                    if (whole) {
                        c.put_row(h, Z, inv, static_cast<T*>(p.out) + (qh0 + head) * D);
                    } else {
                        c.put_row(h, Z, inv, p.partial + (record * p.heads + head) * D);
                        if (lane < 4) p.lse[record * p.heads + head] = L == 0.f ? -INFINITY : c.m[h] + log2f(L);
                    }
                }
            }
            if (!whole) {
                const int c0 = owner(unit_lo), c1 = owner(unit_lo + seg.tiles - 1);
                __syncwarp();  // the ticket's release covers the stores of the warp before it
                unsigned int old = 0;
                if (lane == 0)
                    asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;"
                                 : "=r"(old) : "l"(p.tickets + unit), "r"((unsigned int)(c1 - c0)) : "memory");
                __syncwarp();  // and its acquire the loads of the warp behind it (a shuffle orders no memory)
                if (__shfl_sync(0xffffffffu, old, 0) == (unsigned int)(c1 - c0))
                    join_partials<T, D>(p, unit + c0, c1 - c0 + 1, heads, qh0, lane, 32);
            }
        } else {
            // ---- join the warps: common maximum, then sums in the order of the warps
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float L = column_sum(c.l[h]), Z = column_sum(c.z[h]);
                if (lane < 4) {
                    stats[warp * 8 + 2 * c.q4 + h] = c.m[h];
                    stats[(W + warp) * 8 + 2 * c.q4 + h] = L;
                    stats[(2 * W + warp) * 8 + 2 * c.q4 + h] = Z;
                }
            }
            __syncthreads();
            auto joined_max = [&](int head) {
                float mx = stats[head];
#pragma unroll
                for (int w = 1; w < W; ++w) mx = fmaxf(mx, stats[w * 8 + head]);
                return mx;
            };
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
                f[h] = c.m[h] == -INFINITY ? 0.f : exp2_fast(c.m[h] - joined_max(2 * c.q4 + h));
            for (int h0 = 0; h0 < heads; h0 += 4) {  // four heads at a time
                // warp w sums heads h0 + w, h0 + w + W, ...
                constexpr int PER = (4 + W - 1) / W;
                float inv[PER], zj[PER];
#pragma unroll
                for (int r = 0; r < PER; ++r) {
                    const int head = h0 + warp + r * W;
                    inv[r] = zj[r] = 0.f;
                    if (head < min(heads, h0 + 4)) {
                        const float mx = joined_max(head);
                        float L = 0.f, Z = 0.f;
#pragma unroll
                        for (int w = 0; w < W; ++w) {
                            const float mw = stats[w * 8 + head];
                            const float fw = mw == -INFINITY ? 0.f : exp2_fast(mw - mx);
                            L = fmaf(stats[(W + w) * 8 + head], fw, L);
                            Z = fmaf(stats[(2 * W + w) * 8 + head], fw, Z);
                        }
                        inv[r] = L == 0.f ? 0.f : 1.f / L;
                        zj[r] = Z;
                        if (!whole && lane == 0)
                            p.lse[record * p.heads + head] = L == 0.f ? -INFINITY : mx + log2f(L);
                    }
                }
                for (int u = 0; u < Consumer::kPieces; ++u) {
                    if (u || h0) __syncthreads();
                    if (c.q4 >> 1 == h0 >> 2) c.put_piece(u, f, piece + warp * 128);
                    __syncthreads();
#pragma unroll
                    for (int r = 0; r < PER; ++r) {
                        const int head = h0 + warp + r * W;
                        if (head < min(heads, h0 + 4)) {
                            float sum = zj[r];
#pragma unroll
                            for (int w = 0; w < W; ++w) sum += piece[w * 128 + (head - h0) * 32 + lane];
                            const int d = Consumer::dim_of(u, lane);
                            if (whole)
                                static_cast<T*>(p.out)[(qh0 + head) * D + d] = Elem<T>::from_float(sum * inv[r]);
                            else
                                p.partial[(record * p.heads + head) * D + d] = sum * inv[r];
                        }
                    }
                }
            }
            if (!whole) {
                // ---- the CTA that takes the unit's last ticket joins its partials
                const int c0 = owner(unit_lo), c1 = owner(unit_lo + seg.tiles - 1);
                __syncthreads();  // the ticket's release covers the stores of the CTA before it
                if (tid == 0) {
                    unsigned int old;
                    asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;"
                                 : "=r"(old) : "l"(p.tickets + unit), "r"((unsigned int)(c1 - c0)) : "memory");
                    last_ticket = old == (unsigned int)(c1 - c0);
                }
                __syncthreads();
                if (last_ticket) join_partials<T, D>(p, unit + c0, c1 - c0 + 1, heads, qh0, tid, W * 32);
            }
            __syncthreads();  // stats, piece (the consumers' scratch) and last_ticket are free again
        }
        const int n = end - done;
        done = end;
        if (done < run) advance(seg, n);
    }
}

// ------------------------------------------------------------------ host side
struct PageDecodePlan {
    int grid, smem, chunks, heads;
    int64_t units, ws_lse, ws_bytes;
};

// Shapes and the device only: graph-static.
template <typename Consumer, bool INT4>
static void page_decode_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int sms, PageDecodePlan* plan) {
    using Shape = PageShape<Consumer, INT4>;
    constexpr int smem = Shape::kBytes;
    static_assert(smem <= 227 * 1024 - 512, "does not fit shared memory");
    // 228 KB an SM, of which each block takes 1 KB and its static arrays besides
    const int per_sm = D <= 128 && 2 * (smem + 1024 + 256) <= 228 * 1024 ? 2 : 1;
    const int64_t group = Hq / Hkv;
    plan->chunks = (int)((group + 7) / 8);
    plan->heads = (int)(group < 8 ? group : 8);
    plan->units = B * Hkv * plan->chunks;
    plan->grid = sms * per_sm;
    plan->smem = smem;
    const int64_t records = plan->units + (int64_t)plan->grid * Shape::kWarps;
    plan->ws_lse = (records * plan->heads * 4 + 255) / 256 * 256;
    plan->ws_bytes = plan->ws_lse + records * plan->heads * D * 4;
}

}  // namespace minikv
