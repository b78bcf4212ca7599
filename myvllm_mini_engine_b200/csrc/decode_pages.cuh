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
// of log2 P' = s + log2(step'), so P' <= 1 is what is rounded to fp16, whatever
// the steps are; P = P' / step' stays in fp32.
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
// Bound by the bytes of the pages.  TMA boxes or bulk copies of a page's head
// (1 KB at D = 128, block_size 16) would hit the SM's copy rate of about one per
// 45 ns, 3.4 TB/s over the device, so the copies are per lane.  mma.sync rather
// than tcgen05: the group's few query heads are the N = 8 columns, the operands
// are made in registers, and the tensor pipe is far from its limit.
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
    float* partial;           // [units + grid][heads][D]
    float* lse;               // [units + grid][heads], log2
    unsigned int* tickets;    // [units], zero before and after
    int batch, q_heads, kv_heads, group, chunks, heads;  // heads: query heads of a unit's record, min(group, 8)
    int num_blocks, block_size, width, take;
    uint64_t bs_magic;        // v / block_size = v * bs_magic >> 42 for v < 2^20
    int64_t page_stride;      // bytes of a page (all kv heads)
    int64_t head_stride;      // bytes from one kv head's part of a page to the next
    int64_t row_stride;       // bytes from one token's row to the next
    int min_tiles;            // tiles a CTA takes at least
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

constexpr uint32_t kNibbleMask = 0x000f000fu;  // the low nibbles of two halves
constexpr float kCodeScale = 16777216.f;       // 2^24: a nibble in the low bits of a half is code 2^-24

// ---------------------------------------------------------------- consumers
// Both keep, per warp: m (running maximum, log2), l (lane's part of sum P),
// z (4-bit: lane's part of sum P base'), o (accumulators) of the unit's query
// heads; lane (g, q4) = (lane / 4, lane % 4) holds columns (heads) 2 q4, 2 q4 + 1.

// 4-bit pool, 32 tokens a tile in two slices of 16 (the M rows of K Q^T; one
// maximum and one rescale for both).  Row r < 8 of a slice's MMA is its token
// r / 2 + 4 (r % 2) (+ 8 for r >= 8): a lane's V loads of one instruction then
// are of four neighbouring tokens.  The order of the head dims in a dot product
// is free: lane q4 takes dims q4 D/4 .. of K (whole words of codes) and, for
// V^T (dims are the M rows), lane g dims g D/8 ..: in each four of them nibble
// 0 and 2 are rows g and g + 8 of one MMA and nibble 1 and 3 (16 times larger
// as subnormals) of another.
template <typename T, int D>
struct Int4Consumer {
    static constexpr int TT = 32;
    static constexpr int RB = D / 2;                         // bytes of a row's codes
    static constexpr int kRowBytes = RB;                     // ... staged without padding
    static constexpr int kStageBytes = TT * (2 * RB + 8);    // K codes, V codes, K pairs, V pairs
    static constexpr int NW = D / 32;                        // words of K a lane takes of a row
    static constexpr int NH = D / 32;                        // 16-bit runs of V a lane takes of a row
    static constexpr int kPieces = NH;                       // groups of 32 output dims
    // An fp16 output resolves 2^-11: P' then goes in as two fp16 terms (2^-22).  Next to a bf16
    // output's own rounding of 2^-9 one term (2^-12) is lost, and half of V's MMAs are saved.
    static constexpr bool kTwoTerms = std::is_same<T, __half>::value;

    uint32_t qb[2 * NW][2];
    float o[2 * NH][4];
    float m[2], l[2], z[2], qsum[2], qscale[2];
    int g, q4;

    __device__ void setup(int lane) {
        g = lane >> 2;
        q4 = lane & 3;
    }

    // Q of head g in fp16, scaled by a power of two so that its largest magnitude lies in [1, 2): bf16
    // values keep their bits then, whatever their exponents.
    __device__ void begin(const T* q, int heads, float scale_log2) {
        float f[8 * NW];
        float top = 0.f;
        if (g < heads) {
#pragma unroll
            for (int i = 0; i < 8 * NW; i += 8) {
                Elem<T>::load(*reinterpret_cast<const uint4*>(q + g * D + q4 * (D / 4) + i), f + i);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[i + e]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8 * NW; ++i) f[i] = 0.f;
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // exponent of the largest element, kept where 2^-e and 2^e are both normal
        const int e = (top > 0.f && top < INFINITY) ? min(120, max(-120, (int)((__float_as_uint(top) >> 23) & 255) - 127)) : 0;
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = __half2float(__float2half_rn(f[8 * w + i] * down));
                sum += x[i];
            }
            qb[2 * w][0] = Elem<__half>::pack(x[0], x[4]);
            qb[2 * w][1] = Elem<__half>::pack(x[2], x[6]);
            qb[2 * w + 1][0] = Elem<__half>::pack(x[1], x[5]);
            qb[2 * w + 1][1] = Elem<__half>::pack(x[3], x[7]);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const float up = __uint_as_float((uint32_t)(127 + e) << 23) * scale_log2;
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

    __device__ __forceinline__ void tile(const unsigned char* stage, uint32_t valid, float) {
        const unsigned char* kst = stage;
        const unsigned char* vst = stage + TT * RB;
        const __half2* kp = reinterpret_cast<const __half2*>(stage + 2 * TT * RB);
        const __half2* vp = kp + TT;
        const int row = (g >> 1) + 4 * (g & 1);
        float t[2][4], rinv[2][2], vbase[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r0 = 16 * i + row, r1 = r0 + 8;
            uint32_t k0[NW], k1[NW];
            load_k(kst + r0 * RB + q4 * (RB / 4), k0);
            load_k(kst + r1 * RB + q4 * (RB / 4), k1);
            float lo[4] = {0.f, 0.f, 0.f, 0.f}, hi[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const uint32_t a[4] = {k0[w] & kNibbleMask, k1[w] & kNibbleMask, (k0[w] >> 8) & kNibbleMask,
                                       (k1[w] >> 8) & kNibbleMask};
                mma16816<__half>(lo, a, qb[2 * w][0], qb[2 * w][1]);
                const uint32_t b[4] = {k0[w] & (kNibbleMask << 4), k1[w] & (kNibbleMask << 4),
                                       (k0[w] >> 8) & (kNibbleMask << 4), (k1[w] >> 8) & (kNibbleMask << 4)};
                mma16816<__half>(hi, b, qb[2 * w + 1][0], qb[2 * w + 1][1]);
            }
            const float2 kp0 = __half22float2(kp[r0]), kp1 = __half22float2(kp[r1]);
            const float2 vp0 = __half22float2(vp[r0]), vp1 = __half22float2(vp[r1]);
            const float ks0 = fmaxf(kp0.x, kInt4StepMin) * kCodeScale, ks1 = fmaxf(kp1.x, kInt4StepMin) * kCodeScale;
            const float vs0 = fmaxf(vp0.x, kInt4StepMin), vs1 = fmaxf(vp1.x, kInt4StepMin);
            const float lv0 = __log2f(vs0), lv1 = __log2f(vs1);
            rinv[i][0] = __fdividef(1.f, vs0);
            rinv[i][1] = __fdividef(1.f, vs1);
            vbase[i][0] = vp0.y;
            vbase[i][1] = vp1.y;
            const bool ok0 = (valid >> r0) & 1u, ok1 = (valid >> r1) & 1u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float s0 = fmaf(fmaf(hi[h], 0.0625f, lo[h]), ks0, kp0.y * qsum[h]);
                const float s1 = fmaf(fmaf(hi[h + 2], 0.0625f, lo[h + 2]), ks1, kp1.y * qsum[h]);
                t[i][h] = ok0 ? fmaf(s0, qscale[h], lv0) : -INFINITY;
                t[i][h + 2] = ok1 ? fmaf(s1, qscale[h], lv1) : -INFINITY;
            }
        }
        float alpha[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float mx = column_max(fmaxf(fmaxf(t[0][h], t[0][h + 2]), fmaxf(t[1][h], t[1][h + 2])));
            const float mn = fmaxf(m[h], mx);
            alpha[h] = mn == -INFINITY ? 1.f : exp2_fast(m[h] - mn);
            m[h] = mn;
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[h] *= alpha[h];
                z[h] *= alpha[h];
#pragma unroll
                for (int x = 0; x < 2 * NH; ++x) {
                    o[x][h] *= alpha[h];
                    o[x][h + 2] *= alpha[h];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                p[e] = m[e & 1] == -INFINITY ? 0.f : exp2_fast(t[i][e] - m[e & 1]);
                const float w = p[e] * rinv[i][e >> 1];
                l[e & 1] += w;
                z[e & 1] = fmaf(w, vbase[i][e >> 1], z[e & 1]);
            }
            const uint32_t p01 = Elem<__half>::pack(p[0], p[1]), p23 = Elem<__half>::pack(p[2], p[3]);
            const uint32_t b0 = transpose8x8(p01), b1 = transpose8x8(p23);
            uint32_t c0 = 0, c1 = 0;
            if constexpr (kTwoTerms) {
                float back[4];
                Elem<__half>::unpack(p01, back);
                Elem<__half>::unpack(p23, back + 2);
                c0 = transpose8x8(Elem<__half>::pack(p[0] - back[0], p[1] - back[1]));
                c1 = transpose8x8(Elem<__half>::pack(p[2] - back[2], p[3] - back[3]));
            }
            uint32_t x0[NH], x1[NH];
            const unsigned char* v = vst + (16 * i + q4) * RB + g * (RB / 8);
            load_v(v, v + 4 * RB, x0);
            load_v(v + 8 * RB, v + 12 * RB, x1);
#pragma unroll
            for (int u = 0; u < NH; ++u) {
                const uint32_t a[4] = {x0[u] & kNibbleMask, (x0[u] >> 8) & kNibbleMask, x1[u] & kNibbleMask,
                                       (x1[u] >> 8) & kNibbleMask};
                const uint32_t b[4] = {x0[u] & (kNibbleMask << 4), (x0[u] >> 8) & (kNibbleMask << 4),
                                       x1[u] & (kNibbleMask << 4), (x1[u] >> 8) & (kNibbleMask << 4)};
                mma16816<__half>(o[2 * u], a, b0, b1);
                mma16816<__half>(o[2 * u + 1], b, b0, b1);
                if constexpr (kTwoTerms) {
                    mma16816<__half>(o[2 * u], a, c0, c1);
                    mma16816<__half>(o[2 * u + 1], b, c0, c1);
                }
            }
        }
    }

    // Piece u of the accumulators times f[h]: element [head][x] for x < 32 is output dim dim_of(u, x).
    __device__ __forceinline__ void put_piece(int u, const float* f, float* dst) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float lo = f[h] * kCodeScale, hi = f[h] * (kCodeScale / 16.f);
            *reinterpret_cast<float4*>(dst + (2 * q4 + h) * 32 + 4 * g) =
                make_float4(o[2 * u][h] * lo, o[2 * u + 1][h] * hi, o[2 * u][h + 2] * lo, o[2 * u + 1][h + 2] * hi);
        }
    }
    __device__ static __forceinline__ int dim_of(int u, int x) { return (x >> 2) * (D / 8) + 4 * u + (x & 3); }
};

// 16-bit pool, 16 tokens a tile; K and V rows are padded by 16 bytes so that
// the 8 rows of an ldmatrix meet different banks.  P goes in as two terms of the
// pool's type, as in the decode over whole tables.
template <typename T, int D>
struct Wide16Consumer {
    static constexpr int TT = 16;
    static constexpr int RB = 2 * D;
    static constexpr int kRowBytes = RB + 16;
    static constexpr int kStageBytes = TT * 2 * kRowBytes;
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

    __device__ __forceinline__ void tile(const unsigned char* stage, uint32_t valid, float scale_log2) {
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
        float alpha[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float mn = fmaxf(m[h], column_max(fmaxf(s[h], s[h + 2])));
            alpha[h] = mn == -INFINITY ? 1.f : exp2_fast(m[h] - mn);
            m[h] = mn;
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[h] *= alpha[h];
#pragma unroll
                for (int x = 0; x < KSTEPS; ++x) {
                    o[x][h] *= alpha[h];
                    o[x][h + 2] *= alpha[h];
                }
            }
        }
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            p[e] = m[e & 1] == -INFINITY ? 0.f : exp2_fast(s[e] - m[e & 1]);
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

    __device__ __forceinline__ void put_piece(int u, const float* f, float* dst) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* row = dst + (2 * q4 + h) * 32 + g;
            row[0] = o[2 * u][h] * f[h];
            row[8] = o[2 * u][h + 2] * f[h];
            row[16] = o[2 * u + 1][h] * f[h];
            row[24] = o[2 * u + 1][h + 2] * f[h];
        }
    }
    __device__ static __forceinline__ int dim_of(int u, int x) { return 32 * u + x; }
};

// ------------------------------------------------------------------ the kernel
template <typename Consumer, bool INT4> struct PageShape {
    static constexpr int kWarps = INT4 ? 8 : 4;
    static constexpr int kStages = INT4 ? 2 : 3;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kRing = kWarps * kStages * Consumer::kStageBytes;
    static constexpr int kPiece = kWarps * 8 * 32 * 4;  // one piece of every warp's accumulators
    // ring | piece | warps' (m, l, z) of 8 heads | stage masks | tile prefix
    static constexpr int kFixed = kRing + kPiece + kWarps * 8 * 3 * 4 + kWarps * kStages * 4;
};

// A place in the list of tiles: tile j of unit ul (of request b).
struct TileCursor {
    int b, ul, j, tiles;  // tiles: of each unit of request b
};

template <typename T, int D, typename Consumer, bool INT4, bool SELECTED>
__global__ void __launch_bounds__(PageShape<Consumer, INT4>::kThreads, (INT4 ? D <= 128 : D <= 128) ? 2 : 1)
    page_decode_kernel(const PageDecodeParams p) {
    using Shape = PageShape<Consumer, INT4>;
    constexpr int TT = Consumer::TT, W = Shape::kWarps, NS = Shape::kStages, RB = Consumer::RB;
    extern __shared__ __align__(128) unsigned char smem[];
    float* piece = reinterpret_cast<float*>(smem + Shape::kRing);
    float* stats = reinterpret_cast<float*>(smem + Shape::kRing + Shape::kPiece);  // [3][W][8]
    uint32_t* masks = reinterpret_cast<uint32_t*>(stats + 3 * W * 8);              // [W][NS]
    int* prefix = reinterpret_cast<int*>(masks + W * NS);                          // [B + 1] tiles per unit
    __shared__ int warp_sums[W];
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
    // ---- exclusive prefix of the requests' tile counts
    {
        const int per = (B + W * 32 - 1) / (W * 32);
        const int lo = min(B, tid * per), hi = min(B, lo + per);
        int sum = 0;
        for (int i = lo; i < hi; ++i) {
            const int n = tiles_of(usable(i));
            prefix[i] = n;
            sum += n;
        }
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
        for (int i = lo; i < hi; ++i) {
            const int n = prefix[i];
            prefix[i] = run;
            run += n;
        }
        if (tid == W * 32 - 1) prefix[B] = run;
        __syncthreads();
    }
    // ---- rows of requests with nothing to attend are zeros
    for (int b = blockIdx.x; b < B; b += gridDim.x)
        if (prefix[b + 1] == prefix[b])
            for (int i = tid; i < p.q_heads * D; i += W * 32)
                static_cast<T*>(p.out)[(int64_t)b * p.q_heads * D + i] = Elem<T>::from_float(0.f);
    // ---- this CTA's run of tiles
    const int64_t total = (int64_t)prefix[B] * U;
    const int64_t most = (total + p.min_tiles - 1) / p.min_tiles;
    const int64_t G = most < gridDim.x ? most : gridDim.x;
    if (blockIdx.x >= G) return;
    const int64_t t0 = blockIdx.x * total / G, t1 = (blockIdx.x + 1) * total / G;
    if (t0 >= t1) return;

    auto cursor_at = [&](int64_t t) -> TileCursor {
        const int64_t x = t / U;  // the request whose tiles [prefix * U, ...) hold t
        int lo = 0, hi = B - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] <= x) lo = mid; else hi = mid - 1;
        }
        TileCursor c;
        c.b = lo;
        c.tiles = prefix[lo + 1] - prefix[lo];
        const int in = (int)(t - (int64_t)prefix[lo] * U);
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
                    c.tiles = prefix[c.b + 1] - prefix[c.b];
                } while (c.tiles == 0);
            }
        }
    };

    // ---- the warp's copies.  Two look-ups run ahead of them, each one tile further: the listed block
    // of a token (lane r holds token r of the tile), then its page.
    unsigned char* ring = smem + warp * NS * Consumer::kStageBytes;
    const uint32_t ring_addr = smem_addr(ring);
    uint32_t* my_masks = masks + warp * NS;
    TileCursor ahead = cursor_at(t0);
    int64_t t_list = t0 + warp;  // the next tile to look up
    if (t_list < t1) advance(ahead, warp);
    int64_t list_block = -1;     // listed block, and where the token lies
    int list_off = 0, list_b = 0, list_kvh = 0, list_len = 0, len_b = -1, len_now = 0;
    int page = -1, page_off = 0, page_kvh = 0;
    int64_t t_copy = t0 + warp;  // the next tile to copy

    auto look_block = [&]() {
        list_block = -1;
        if (t_list < t1) {
            if (ahead.b != len_b) {
                len_b = ahead.b;
                len_now = usable(len_b);
            }
            list_b = ahead.b;
            list_len = len_now;
            list_kvh = ahead.ul / p.chunks;
            const int v = ahead.j * TT + (TT == 32 ? lane : lane & 15);
            const int e = (int)(((uint64_t)v * p.bs_magic) >> 42);
            list_off = v - e * p.block_size;
            if (SELECTED) {
                if (e < p.take) list_block = p.selected[((int64_t)list_b * p.kv_heads + list_kvh) * p.take + e];
            } else {
                list_block = e;
            }
            t_list += W;
            if (t_list < t1) advance(ahead, W);
        }
    };
    auto look_page = [&]() {
        page = -1;
        page_off = list_off;
        page_kvh = list_kvh;
        if (list_block >= 0 && list_block < p.width && list_block * p.block_size + list_off < list_len) {
            const int64_t id = p.tables[(int64_t)list_b * p.width + list_block];
            page = id >= 0 && id < p.num_blocks ? (int)id : -1;
        }
    };
    auto copy_tile = [&](int slot) {
        if (t_copy < t1) {
            const uint32_t dst = ring_addr + slot * Consumer::kStageBytes;
            const uint32_t valid = __ballot_sync(0xffffffffu, page >= 0);
            if (lane == 0) my_masks[slot] = valid;
            const int64_t head = (int64_t)page_kvh * p.head_stride;
            constexpr int CPR = RB / 16;  // 16-byte pieces of a row
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
                const int64_t at =
                    page < 0 ? 0 : page * p.page_stride + head + (int64_t)p.block_size * RB + page_off * 4;
                copy4(dst + 2 * TT * RB + lane * 4, p.kc + at, page < 0 ? 0u : 4u);
                copy4(dst + 2 * TT * RB + TT * 4 + lane * 4, p.vc + at, page < 0 ? 0u : 4u);
            }
            t_copy += W;
        }
        copy_commit();
    };
    look_block();
    look_page();
    look_block();
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
        copy_tile(s);
        look_page();
        look_block();
    }

    Consumer c;
    c.setup(lane);
    int slot = 0;
    int64_t t = t0 + warp;
    TileCursor seg = cursor_at(t0);
    for (int64_t lo = t0; lo < t1;) {
        // ---- one unit's tiles in this CTA's run: [lo, hi)
        const int64_t unit_lo = (int64_t)prefix[seg.b] * U + (int64_t)seg.ul * seg.tiles, unit_hi = unit_lo + seg.tiles;
        const int64_t hi = unit_hi < t1 ? unit_hi : t1;
        const int kvh = seg.ul / p.chunks, chunk = seg.ul - kvh * p.chunks;
        const int heads = min(8, p.group - 8 * chunk);
        const int64_t qh0 = (int64_t)seg.b * p.q_heads + kvh * p.group + 8 * chunk;
        c.begin(static_cast<const T*>(p.q) + qh0 * D, heads, p.scale_log2);
        for (; t < hi; t += W) {
            copy_wait<NS - 2>();
            __syncwarp();  // the stage is whole, and the one filled next has been read by every lane
            copy_tile(slot == 0 ? NS - 1 : slot - 1);
            look_page();
            look_block();
            c.tile(ring + slot * Consumer::kStageBytes, my_masks[slot], p.scale_log2);
            slot = slot + 1 == NS ? 0 : slot + 1;
        }
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
        for (int h = 0; h < 2; ++h) {
            const float mx = joined_max(2 * c.q4 + h);
            f[h] = c.m[h] == -INFINITY ? 0.f : exp2_fast(c.m[h] - mx);
        }
        const bool whole = lo == unit_lo && hi == unit_hi;
        const int64_t unit = (int64_t)seg.b * U + seg.ul;
        const int64_t record = unit + blockIdx.x;  // grows by at least one from segment to segment
        // W * 32 threads sum 8 x 32 elements a piece
        constexpr int PER = 256 / (W * 32);
        float inv[PER], zj[PER];
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const int head = (tid + r * W * 32) >> 5;
            const float mx = joined_max(head);
            float L = 0.f, Z = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float mw = stats[w * 8 + head];
                const float fw = mw == -INFINITY ? 0.f : exp2_fast(mw - mx);
                L = fmaf(stats[(W + w) * 8 + head], fw, L);
                Z = fmaf(stats[(2 * W + w) * 8 + head], fw, Z);
            }
            inv[r] = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);  // NaN stays
            zj[r] = Z;
            if (!whole && lane == 0 && head < heads)
                p.lse[record * p.heads + head] = L == 0.f ? -INFINITY : mx + log2f(L);
        }
        for (int u = 0; u < Consumer::kPieces; ++u) {
            if (u) __syncthreads();
            c.put_piece(u, f, piece + warp * 256);
            __syncthreads();
#pragma unroll
            for (int r = 0; r < PER; ++r) {
                const int head = (tid + r * W * 32) >> 5;
                if (head < heads) {
                    float sum = zj[r];
#pragma unroll
                    for (int w = 0; w < W; ++w) sum += piece[w * 256 + head * 32 + lane];
                    const int d = Consumer::dim_of(u, lane);
                    if (whole)
                        static_cast<T*>(p.out)[(qh0 + head) * D + d] = Elem<T>::from_float(sum * inv[r]);
                    else
                        p.partial[(record * p.heads + head) * D + d] = sum * inv[r];
                }
            }
        }
        if (!whole) {
            // ---- the CTA that takes the unit's last ticket joins its partials
            auto owner = [&](int64_t x) { return (int)(((x + 1) * G + total - 1) / total) - 1; };
            const int c0 = owner(unit_lo), c1 = owner(unit_hi - 1);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                unsigned int old;
                asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;"
                             : "=r"(old) : "l"(p.tickets + unit), "r"((unsigned int)(c1 - c0)) : "memory");
                last_ticket = old == (unsigned int)(c1 - c0);
            }
            __syncthreads();
            if (last_ticket) {
                __threadfence();
                const int n = c1 - c0 + 1;
                const int64_t first = unit + c0;
                for (int x = tid; x < heads * D; x += W * 32) {
                    const int head = x / D, d = x - head * D;
                    const float* lse = p.lse + first * p.heads + head;
                    const float* part = p.partial + (first * p.heads + head) * D + d;
                    float mx = -INFINITY, sum = 0.f, acc = 0.f;
                    for (int k0 = 0; k0 < n; k0 += 8) {
                        float e[8], v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const bool in = k0 + k < n;
                            e[k] = in ? __ldcg(lse + (int64_t)(k0 + k) * p.heads) : -INFINITY;
                            v[k] = in ? __ldcg(part + (int64_t)(k0 + k) * p.heads * D) : 0.f;
                        }
                        float top = mx;
#pragma unroll
                        for (int k = 0; k < 8; ++k) top = fmaxf(top, e[k]);
                        const float keep = mx == -INFINITY ? 0.f : exp2_fast(mx - top);
                        sum *= keep;
                        acc *= keep;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float w = e[k] == -INFINITY ? 0.f : exp2_fast(e[k] - top);
                            sum += w;
                            acc = fmaf(w, v[k], acc);
                        }
                        mx = top;
                    }
                    static_cast<T*>(p.out)[(qh0 + head) * D + d] =
                        Elem<T>::from_float(sum == 0.f ? 0.f : acc / sum);
                }
            }
        }
        __syncthreads();  // stats, piece and last_ticket are free again
        advance(seg, (int)(hi - lo));
        lo = hi;
    }
}

// ------------------------------------------------------------------ host side
struct PageDecodePlan {
    int grid, smem, chunks, heads;
    int64_t units, ws_lse, ws_partial, ws_bytes;
};

// Shapes and the device only: graph-static.
template <typename Consumer, bool INT4>
static bool page_decode_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int sms, PageDecodePlan* plan) {
    using Shape = PageShape<Consumer, INT4>;
    const int64_t smem = Shape::kFixed + (B + 1) * 4;
    if (smem > 227 * 1024 - 1024) return false;
    const int per_sm = D <= 128 && 2 * (smem + 2048) <= 227 * 1024 ? 2 : 1;
    const int64_t group = Hq / Hkv;
    plan->chunks = (int)((group + 7) / 8);
    plan->heads = (int)(group < 8 ? group : 8);
    plan->units = B * Hkv * plan->chunks;
    plan->grid = sms * per_sm;
    plan->smem = (int)smem;
    const int64_t records = plan->units + plan->grid;
    plan->ws_lse = (records * plan->heads * 4 + 255) / 256 * 256;
    plan->ws_partial = 0;
    plan->ws_bytes = plan->ws_lse + records * plan->heads * D * 4;
    return true;
}

}  // namespace minikv
