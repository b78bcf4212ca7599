// Ragged causal prefill over a 4-bit pool.
//
// Packed query token i of request r sits at position start + i and attends the
// keys [0, start + i] of r's pages (history and current chunk, already written).
// A CTA takes 64 rows, (token, query head) pairs of one request and kv head, 16
// a warp, and goes over the keys BN at a time with a running maximum and sum:
//   S = Q K^T,  s = (step (q . c) + base sum(q)) / sqrt(D),  P' = 2^(s + log2 step' - max)
//   O += P' C'^T,  l += P' / step',  z += P' base' / step',  out = (O + z) / l
// As in decode_pages.cuh the codes are the operands, nibbles masked out of the
// staged words (fp16 subnormals c 2^-24, c 2^-20; Q of the latter is scaled by
// 1/16 beforehand, so one accumulator serves both).  The maximum is a
// row's own, of s + log2 step' over the keys that it sees: keys of no weight, or
// behind the row, do not move what its P' is rounded to, whatever their steps.
// P' enters in two fp16 terms (2^-22): one (2^-12) would move half of an fp16
// output's roundings to the next value, and a twentieth of a bf16 one's (4 x 1000
// tokens behind 4096, 32/8 heads of 128: 1181 us with one term, 1515 with two).
// O of a tile of keys is summed by itself and then added (the same: 1473 us with
// MMAs that add to the row's, 1593 so).
//
// Bound by the tensor pipe (48 % of its cycles), by issue (40 %) and by the
// latencies that 8 warps a SM leave open: a warp makes its operands from the codes
// itself.  mma.sync rather than tcgen05: a tcgen05 operand has to lie in
// shared memory as 16-bit values, four times the codes' bytes written there and
// read back per tile, while the masked registers feed mma.sync as they are and
// the P operand never leaves them.
#pragma once

#include "decode_pages.cuh"

namespace minikv {

struct PrefillInt4Params {
    const void* q;
    const unsigned char* kc;
    const unsigned char* vc;
    const int64_t* cu;
    const int64_t* starts;
    const int64_t* tables;
    const int64_t* lens;
    void* out;
    int64_t tokens, width, num_blocks, page_bytes;
    int requests, q_heads, kv_heads, group, block_size, tile_tokens;  // tile_tokens: 64 / group
    uint64_t bs_magic;
    float scale_log2;
};

constexpr int kPrefillWarps = 4;
constexpr int kPrefillThreads = kPrefillWarps * 32;
constexpr int kPrefillRows = kPrefillWarps * 16;
constexpr int kPrefillStages = 3;

// N (1, 2 or 4) 16-bit runs of the rows of two keys, side by side (the first key's in the low half)
template <int N>
__device__ __forceinline__ void load_value_runs(const unsigned char* a, const unsigned char* b, uint32_t* x) {
    if constexpr (N == 1) {
        x[0] = *reinterpret_cast<const uint16_t*>(a) | ((uint32_t) * reinterpret_cast<const uint16_t*>(b) << 16);
    } else {
        uint32_t wa[N / 2], wb[N / 2];
        if constexpr (N == 4) {
            const uint2 c = *reinterpret_cast<const uint2*>(a), d = *reinterpret_cast<const uint2*>(b);
            wa[0] = c.x; wa[1] = c.y;
            wb[0] = d.x; wb[1] = d.y;
        } else {
            wa[0] = *reinterpret_cast<const uint32_t*>(a);
            wb[0] = *reinterpret_cast<const uint32_t*>(b);
        }
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            x[2 * i] = permute_bytes(wa[i], wb[i], 0x5410u);
            x[2 * i + 1] = permute_bytes(wa[i], wb[i], 0x7632u);
        }
    }
}

// CTAs a SM: three at 64 dims or fewer (4 x 1000 tokens behind 4096, 32/8 heads of 64: 916 us, with two
// 992; though 32 x 8 behind 2048, 16/8 heads, 92 and 69); at 96 and 128 the registers of three spill, and two
// take 1592 against 1645 us at 128, and 32 x 8 tokens 108 against 166.
template <typename T, int D>
__global__ void __launch_bounds__(kPrefillThreads, D <= 64 ? 3 : 2) prefill_int4_kernel(const PrefillInt4Params p) {
    constexpr int BN = D <= 128 ? 64 : 32;  // keys a tile: the accumulators of S take BN / 2 registers
    constexpr int RB = D / 2, CPR = RB / 16, NW = D / 32, NT = BN / 8;
    constexpr int NV = NW % 4 == 0 ? 4 : NW % 2 == 0 ? 2 : 1;  // 16-bit runs of V a lane loads at once, of NW (registers)
    constexpr int STAGE = BN * (2 * RB + 8);  // K codes, V codes, K pairs, V pairs
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q4 = lane & 3;
    __shared__ __align__(128) unsigned char ring[kPrefillStages * STAGE];
    __shared__ int64_t row_at[2][BN];     // byte of a key's codes in the pool, or -1
    __shared__ int64_t pair_at[2][BN];
    __shared__ uint32_t valid_s[kPrefillStages][2];
    // of the keys of a tile, by each warp for itself: K step 2^24, K base, log2 V step, 1 / V step; V base / V step
    __shared__ float4 factors_s[kPrefillWarps][BN];
    __shared__ float weights_s[kPrefillWarps][BN];
    float4* factors = factors_s[warp];
    float* weights = weights_s[warp];
    const int kvh = blockIdx.x, r = blockIdx.z;
    griddep_wait();
    griddep_launch_dependents();
    const int64_t cu0 = p.cu[r], cu1 = p.cu[r + 1], start = p.starts[r], len = p.lens[r];
    const int64_t* table = p.tables + (int64_t)r * p.width;
    T* out = static_cast<T*>(p.out);
    // ---- packed tokens of no request get zeros
    if (r == 0 || r == p.requests - 1) {
        const int64_t heads = p.group * D;
        auto zero = [&](int64_t a, int64_t b) {
            a = a < 0 ? 0 : a;
            b = b > p.tokens ? p.tokens : b;
            for (int64_t x = (int64_t)blockIdx.y * kPrefillThreads + tid; x < (b - a) * heads;
                 x += (int64_t)gridDim.y * kPrefillThreads)
                out[((a + x / heads) * p.q_heads + (int64_t)kvh * p.group) * D + x % heads] = Elem<T>::from_float(0.f);
        };
        if (r == 0) zero(0, cu0);
        if (r == p.requests - 1) zero(cu1, p.tokens);
    }
    if (cu0 < 0 || cu1 > p.tokens || cu0 >= cu1) return;
    const int64_t count = cu1 - cu0;
    const int64_t tiles = (count + p.tile_tokens - 1) / p.tile_tokens;
    const int64_t reach = min(len, p.width * (int64_t)p.block_size);  // keys that exist

    // the latest tiles, which see the most keys, come first
    for (int64_t qt = tiles - 1 - blockIdx.y; qt >= 0; qt -= gridDim.y) {
        const int64_t i0 = qt * p.tile_tokens;
        const int here = (int)min((int64_t)p.tile_tokens, count - i0);  // tokens of this tile
        // ---- rows of this lane: warp * 16 + g and + 8
        int64_t row_out[2];
        int last[2];  // last visible key of the row, -1: none
        uint32_t qa[2 * NW][4];
        float qsum[2], qscale[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int row = warp * 16 + g + 8 * x;
            const int tok = row / p.group, hd = row - tok * p.group;
            const bool in = tok < here;
            row_out[x] = in ? ((cu0 + i0 + tok) * p.q_heads + (int64_t)kvh * p.group + hd) * D : -1;
            const int64_t pos = start + i0 + tok;
            last[x] = in && pos >= 0 && pos < reach ? (int)pos : -1;
            float f[8 * NW];
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8 * NW; i += 8) {
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (in) v = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + row_out[x] + q4 * (D / 4) + i);
                Elem<T>::load(v, f + i);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[i + e]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e2 = query_exponent(top);  // scaled as in the decode
            const float down = power_of_two(-e2);
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    // the operand of a high nibble, 16 times larger as a subnormal
                    const float unit = (i & 1) ? 0.0625f : 1.f;
                    y[i] = __half2float(__float2half_rn(f[8 * w + i] * down * unit));
                    sum += (i & 1) ? y[i] * 16.f : y[i];
                }
                qa[2 * w][x] = Elem<__half>::pack(y[0], y[4]);
                qa[2 * w][2 + x] = Elem<__half>::pack(y[2], y[6]);
                qa[2 * w + 1][x] = Elem<__half>::pack(y[1], y[5]);
                qa[2 * w + 1][2 + x] = Elem<__half>::pack(y[3], y[7]);
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            qsum[x] = sum;
            qscale[x] = power_of_two(e2) * p.scale_log2;
        }
        // a row past the context sees nothing, whatever its neighbours see
        const bool odd_rows = __any_sync(0xffffffffu, (row_out[0] >= 0 && last[0] < 0) || (row_out[1] >= 0 && last[1] < 0));
        // ---- keys this tile sees, and those that all of the warp's rows see
        const int64_t far = start + i0 + here - 1;
        const int keys = (int)max((int64_t)0, min(reach, far + 1));
        const int warp_near = (int)max((int64_t)0, min(reach, start + i0 + (warp * 16) / p.group + 1));
        const int nk = (keys + BN - 1) / BN;

        auto look = [&](int kt) {  // threads below BN: where the tile's keys lie
            if (tid < BN) {
                const int pos = kt * BN + tid;
                int64_t at = -1, pair = -1;
                if (pos < keys) {
                    const int e = (int)(((uint64_t)pos * p.bs_magic) >> 42);
                    const int64_t page = table[e];
                    if (page >= 0 && page < p.num_blocks) {
                        const int off = pos - e * p.block_size;
                        const int64_t base = (page * p.kv_heads + kvh) * p.page_bytes;
                        at = base + (int64_t)off * RB;
                        pair = base + (int64_t)p.block_size * RB + off * 4;
                    }
                }
                row_at[kt & 1][tid] = at;
                pair_at[kt & 1][tid] = pair;
            }
        };
        auto copy = [&](int kt) {
            if (kt < nk) {
                const int s = kt % kPrefillStages;
                const uint32_t dst = smem_addr(ring) + s * STAGE;
#pragma unroll
                for (int c0 = 0; c0 < BN * CPR; c0 += kPrefillThreads) {
                    const int c = c0 + tid;
                    if (BN * CPR % kPrefillThreads == 0 || c < BN * CPR) {
                        const int row = c / CPR, x = c - row * CPR;
                        const int64_t at = row_at[kt & 1][row];
                        const int64_t from = at < 0 ? 0 : at + x * 16;
                        const uint32_t n = at < 0 ? 0u : 16u;
                        copy16(dst + row * RB + x * 16, p.kc + from, n);
                        copy16(dst + (BN + row) * RB + x * 16, p.vc + from, n);
                    }
                }
                if (tid < 2 * BN) {
                    const int64_t at = pair_at[kt & 1][tid % BN];
                    copy4(dst + 2 * BN * RB + tid * 4, (tid < BN ? p.kc : p.vc) + (at < 0 ? 0 : at), at < 0 ? 0u : 4u);
                }
                if (tid < BN) {
                    const uint32_t bits = __ballot_sync(0xffffffffu, row_at[kt & 1][tid] >= 0);
                    if (lane == 0) valid_s[s][warp] = bits;
                }
            }
            copy_commit();
        };
        __syncthreads();  // the ring and the look-ups of the tile before are free
        look(0);
        __syncthreads();
        copy(0);
        look(1);
        __syncthreads();
        copy(1);
        // (the loop's first barrier comes before look(2) is needed)

        float o[NW][4][4];
#pragma unroll
        for (int u = 0; u < NW; ++u)
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[u][n][i] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, z[2] = {0.f, 0.f};

        for (int kt = 0; kt < nk; ++kt) {
            copy_wait<1>();
            look(kt + 2);     // the look-ups of tile kt, whose buffer this takes, were used by copy(kt)
            __syncthreads();  // tile kt is whole; every warp is done with tile kt - 1
            copy(kt + 2);
            const unsigned char* st = ring + (kt % kPrefillStages) * STAGE;
            const uint64_t valid = valid_s[kt % kPrefillStages][0] |
                                   (BN > 32 ? (uint64_t)valid_s[kt % kPrefillStages][1] << 32 : 0ull);
            const __half2* pairs = reinterpret_cast<const __half2*>(st + 2 * BN * RB);
#pragma unroll
            for (int i = 0; i < BN / 32; ++i) {
                const float2 k = __half22float2(pairs[32 * i + lane]), v = __half22float2(pairs[BN + 32 * i + lane]);
                const float vstep = fmaxf(v.x, kInt4StepMin);
                const float inv = rcp_fast(vstep);
                factors[32 * i + lane] = make_float4(fmaxf(k.x, kInt4StepMin) * kCodeScale, k.y, log2_fast(vstep), inv);
                weights[32 * i + lane] = v.y * inv;
            }
            __syncwarp();
            // ---- S: column c of key group j is its key c / 2 + 4 (c % 2)
            float s[NT][4];
#pragma unroll
            for (int j = 0; j < NT; j += 2) {  // two groups at a time: their MMA chains overlap
                uint32_t w[2][NW];
#pragma unroll
                for (int jj = 0; jj < 2; ++jj) {
                    const unsigned char* src = st + (8 * (j + jj) + (g >> 1) + 4 * (g & 1)) * RB + q4 * (RB / 4);
                    if constexpr (NW % 4 == 0) {
#pragma unroll
                        for (int i = 0; i < NW / 4; ++i) {
                            const uint4 v = *reinterpret_cast<const uint4*>(src + 16 * i);
                            w[jj][4 * i] = v.x; w[jj][4 * i + 1] = v.y; w[jj][4 * i + 2] = v.z; w[jj][4 * i + 3] = v.w;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < NW; ++i) w[jj][i] = *reinterpret_cast<const uint32_t*>(src + 4 * i);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[j + jj][i] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < NW; ++i) {
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj)
                        mma16816<__half>(s[j + jj], qa[2 * i], w[jj][i] & kNibbleMask, (w[jj][i] >> 8) & kNibbleMask);
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj)
                        mma16816<__half>(s[j + jj], qa[2 * i + 1], w[jj][i] & (kNibbleMask << 4),
                                         (w[jj][i] >> 8) & (kNibbleMask << 4));
                }
            }
            // ---- scores and their maxima
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float4 f = factors[8 * j + q4 + 4 * y];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float& e = s[j][2 * x + y];
                        e = fmaf(fmaf(e, f.x, f.y * qsum[x]), qscale[x], f.z);
                    }
                }
            if (odd_rows || (kt + 1) * BN > warp_near || valid != (BN == 64 ? ~0ull : 0xffffffffull)) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = 8 * j + q4 + 4 * (i & 1);
                        if (kt * BN + key > last[i >> 1] || !((valid >> key) & 1ull)) s[j][i] = -INFINITY;
                    }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx[i >> 1] = fmaxf(mx[i >> 1], s[j][i]);
            if (__any_sync(0xffffffffu, mx[0] > m[0] + kMost || mx[1] > m[1] + kMost)) {
                float alpha[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
                    mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
                    const float mn = mx[x] > m[x] + kMost ? mx[x] - kHeadroom : m[x];
                    alpha[x] = mn == -INFINITY ? 1.f : exp2_fast(m[x] - mn);
                    m[x] = mn;
                    l[x] *= alpha[x];
                    z[x] *= alpha[x];
                }
#pragma unroll
                for (int u = 0; u < NW; ++u)
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[u][n][i] *= alpha[i >> 1];
            }
            // ---- P' as the A operands
            const float mm[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
            uint32_t a[NT / 2][4], a2[NT / 2][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float inv[2], base[2];  // of the two keys: 1 / V step, V base / V step
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    inv[y] = factors[8 * j + q4 + 4 * y].w;
                    base[y] = weights[8 * j + q4 + 4 * y];
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float w[2], back[2];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        w[y] = exp2_fast(s[j][2 * x + y] - mm[x]);
                        l[x] = fmaf(w[y], inv[y], l[x]);
                        z[x] = fmaf(w[y], base[y], z[x]);
                    }
                    uint32_t& hi = a[j / 2][2 * (j & 1) + x];
                    hi = Elem<__half>::pack(w[0], w[1]);
                    Elem<__half>::unpack(hi, back);
                    a2[j / 2][2 * (j & 1) + x] = Elem<__half>::pack(w[0] - back[0], w[1] - back[1]);
                }
            }
            // ---- O of the tile by itself, then added: an MMA truncates its sum, which the codes (none
            // negative) would turn into a bias that grows with the keys
            uint32_t v[NT / 2][2][NV];
#pragma unroll
            for (int u = 0; u < NW; ++u) {
                if (u % NV == 0) {
#pragma unroll
                    for (int j = 0; j < NT / 2; ++j)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const unsigned char* at = st + (BN + 16 * j + 8 * half + q4) * RB + g * (RB / 8) + 2 * u;
                            load_value_runs<NV>(at, at + 4 * RB, v[j][half]);
                        }
                }
                float d[4][4];
#pragma unroll
                for (int j = 0; j < NT / 2; ++j) {
                    // even nibbles, and whole bytes for the odd ones (as the decode)
                    const uint32_t v0 = v[j][0][u % NV], v1 = v[j][1][u % NV];
                    const uint32_t l0 = v0 & 0x00ff00ffu, l1 = v1 & 0x00ff00ffu;
                    const uint32_t h0 = permute_bytes(v0, 0u, 0x4341u), h1 = permute_bytes(v1, 0u, 0x4341u);
                    const uint32_t b[4][2] = {{l0 & kNibbleMask, l1 & kNibbleMask}, {l0, l1},
                                              {h0 & kNibbleMask, h1 & kNibbleMask}, {h0, h1}};
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        if (j == 0) mma16816_first(d[n], a[j], b[n][0], b[n][1]);
                        else mma16816<__half>(d[n], a[j], b[n][0], b[n][1]);
                    }
#pragma unroll
                    for (int n = 0; n < 4; ++n) mma16816<__half>(d[n], a2[j], b[n][0], b[n][1]);
                }
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[u][n][i] += d[n][i];
            }
        }
        copy_wait<0>();
        // ---- output: lane q4 holds dims [c D/8, (c + 1) D/8) for c = 2 q4 and 2 q4 + 1
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float L = l[x], Z = z[x];
            L += __shfl_xor_sync(0xffffffffu, L, 1);
            L += __shfl_xor_sync(0xffffffffu, L, 2);
            Z += __shfl_xor_sync(0xffffffffu, Z, 1);
            Z += __shfl_xor_sync(0xffffffffu, Z, 2);
            if (row_out[x] < 0) continue;  // no shuffle of this row follows
            const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                T* dst = out + row_out[x] + (2 * q4 + y) * (D / 8);
#pragma unroll
                for (int u = 0; u < NW; ++u) {
                    const int i = 2 * x + y;
                    const float f0 = fmaf(o[u][0][i], kCodeScale, Z) * inv, f2 = fmaf(o[u][2][i], kCodeScale, Z) * inv;
                    const float f1 = fmaf(o[u][1][i] - o[u][0][i], kCodeScale * 0.0625f, Z) * inv;
                    const float f3 = fmaf(o[u][3][i] - o[u][2][i], kCodeScale * 0.0625f, Z) * inv;
                    *reinterpret_cast<uint2*>(dst + 4 * u) = make_uint2(Elem<T>::pack(f0, f1), Elem<T>::pack(f2, f3));
                }
            }
        }
    }
}

}  // namespace minikv
