// Ragged prefill over a 4-bit pool on the tcgen05 kernel, by way of an fp16 copy.
//
// spread_table_pages_kernel writes the pages that the batch reads as dense fp16
// pages (table entry e = r * W + j becomes page e of the copy), a table of them
// (-1 where the entry is no page of the pool or lies past the request's
// context) and Q in fp16; the 16-bit prefill then runs on those, with a bf16
// output.  base + step * code is rounded to fp16 once, 2^-12 relative: under the
// bf16 output's own 2^-9, which is why fp16 outputs do not take this route.  Q
// outside fp16's range is saturated, and below 2^-14 loses bits, as over an FP8
// pool.  It costs four times the pool's bytes written and read again, so it is
// taken from kInt4DenseRows (token, query head) rows a request and kv head.
#include "common.cuh"
#include "int4_pool.cuh"

namespace minikv {

// One CTA an entry of the tables; D / 8 lanes a row of a page, 8 elements each.
template <int D>
__global__ void __launch_bounds__(256) spread_table_pages_kernel(
    const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc, const int64_t* __restrict__ tables,
    const int64_t* __restrict__ lens, const int64_t* __restrict__ cu, int64_t requests, int64_t width,
    int64_t num_blocks, FastDiv block_of, int kv_heads, __half* __restrict__ kout, __half* __restrict__ vout,
    int64_t* __restrict__ new_tables, const __nv_bfloat16* __restrict__ q, __half* __restrict__ qout,
    int64_t q_eights, __nv_bfloat16* __restrict__ out, int64_t token_eights) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int LANES = D / 8;
    const int block_size = (int)block_of.d;
    const int64_t page_bytes = int4_page_bytes(block_size, D);
    const int64_t row_elems = (int64_t)kv_heads * D;
    const int in = threadIdx.x % LANES;
    // ---- pages: K's rows head by head, then V's
    for (int64_t e = blockIdx.x; e < requests * width; e += gridDim.x) {
        const int64_t r = e / width, j = e - r * width;
        const int64_t page = tables[e], left = lens[r] - j * block_size;
        const bool used = page >= 0 && page < num_blocks && left > 0;
        if (threadIdx.x == 0) new_tables[e] = used ? e : -1;
        if (!used) continue;
        const uint32_t rows = 2u * kv_heads * block_size;
#pragma unroll 4
        for (uint32_t row = threadIdx.x / LANES; row < rows; row += 256 / LANES) {
            const uint32_t hv = block_of(row);
            const int t = (int)(row - hv * block_size);
            const bool is_v = hv >= (uint32_t)kv_heads;
            const int h = (int)hv - (is_v ? kv_heads : 0);
            if (t >= left) continue;
            const unsigned char* src = (is_v ? vc : kc) + (page * kv_heads + h) * page_bytes;
            const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(src + t * (D / 2) + in * 4));
            const float2 sb = __half22float2(
                *reinterpret_cast<const __half2*>(src + (int64_t)block_size * (D / 2) + t * 4));
            const float s = fmaxf(sb.x, kInt4StepMin);
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)  // (a rounded pair can reach a little over the largest fp16)
                f[i] = fminf(fmaf(s, (float)((word >> (4 * i)) & 15u), sb.y), 65504.f);
            *reinterpret_cast<uint4*>((is_v ? vout : kout) + (e * block_size + t) * row_elems + h * D + in * 8) =
                Elem<__half>::store(f);
        }
    }
    // ---- packed tokens of no request get zeros, which the prefill leaves as they are
    const int64_t first = max((int64_t)0, cu[0]) * token_eights, behind = max((int64_t)0, cu[requests]) * token_eights;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < q_eights; x += (int64_t)gridDim.x * 256)
        if (x < first || x >= behind) reinterpret_cast<uint4*>(out)[x] = make_uint4(0u, 0u, 0u, 0u);
    // ---- Q
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < q_eights; x += (int64_t)gridDim.x * 256) {
        float f[8];
        Elem<__nv_bfloat16>::load(reinterpret_cast<const uint4*>(q)[x], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = isnan(f[i]) ? f[i] : fminf(fmaxf(f[i], -65504.f), 65504.f);
        reinterpret_cast<uint4*>(qout)[x] = Elem<__half>::store(f);
    }
}

constexpr int64_t kInt4DenseLimit = 8ll << 30;
constexpr int64_t kInt4DenseRows = 128;  // (token, query head) rows a request and kv head, on average

struct Int4DensePlan {
    int64_t value, tables, q, bytes;  // offsets of the parts in the workspace (keys come first)
};

// Whether a batch takes this route, and its workspace.
static bool int4_dense_plan(int64_t tokens, int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                            int64_t block_size, int64_t width, int dtype, Int4DensePlan* plan) {
    const int64_t entries = requests * width;
    if (dtype != MINIKV_BF16 || entries <= 0 || tokens * (q_heads / kv_heads) < kInt4DenseRows * requests ||
        !prefill_tc_supported(q_heads, kv_heads, head_dim, block_size, dtype, entries, tokens, requests))
        return false;
    const int64_t copy = align256(entries * block_size * kv_heads * head_dim * 2);
    plan->value = copy;
    plan->tables = 2 * copy;
    plan->q = plan->tables + align256(entries * 8);
    plan->bytes = plan->q + align256(tokens * q_heads * head_dim * 2);
    return plan->bytes <= kInt4DenseLimit;
}

}  // namespace minikv

extern "C" {

// Bytes of the dense route's workspace, or -1 where a batch does not take it.
__attribute__((visibility("hidden"))) int64_t minikv_prefill_int4_dense_bytes(
    int64_t tokens, int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t block_size,
    int64_t width, int dtype) {
    Int4DensePlan plan;
    return int4_dense_plan(tokens, requests, q_heads, kv_heads, head_dim, block_size, width, dtype, &plan) ? plan.bytes
                                                                                                            : -1;
}

__attribute__((visibility("hidden"))) int minikv_prefill_int4_dense(
    const void* q, const void* key_cache, const void* value_cache, const int64_t* cu, const int64_t* starts,
    const int64_t* tables, const int64_t* lens, void* out, void* workspace, int64_t tokens, int64_t requests,
    int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks, int64_t block_size, int64_t width,
    int dtype, void* stream) {
    Int4DensePlan plan;
    if (!int4_dense_plan(tokens, requests, q_heads, kv_heads, head_dim, block_size, width, dtype, &plan))
        return fail(MINIKV_EUNSUPPORTED, "this 4-bit prefill has no dense route");
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    int64_t* new_tables = reinterpret_cast<int64_t*>(ws + plan.tables);
    const int64_t entries = requests * width;
    const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(entries, (int64_t)sm_count() * 8));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto spread = head_dim == 64 ? spread_table_pages_kernel<64> : spread_table_pages_kernel<128>;
    const cudaError_t err = launch_chained(
        spread, dim3(grid), dim3(256), 0, s, static_cast<const unsigned char*>(key_cache),
        static_cast<const unsigned char*>(value_cache), tables, lens, cu, requests, width, num_blocks,
        FastDiv((uint32_t)block_size), (int)kv_heads, reinterpret_cast<__half*>(ws), reinterpret_cast<__half*>(ws + plan.value), new_tables,
        static_cast<const __nv_bfloat16*>(q), reinterpret_cast<__half*>(ws + plan.q), tokens * q_heads * head_dim / 8,
        static_cast<__nv_bfloat16*>(out), q_heads * head_dim / 8);
    if (err != cudaSuccess) return cuda_fail(err, "minikv_paged_prefill_int4 page spreading");
    return run_prefill_tc(ws + plan.q, ws, ws + plan.value, cu, starts, new_tables, lens, out, tokens, requests, q_heads,
                          kv_heads, head_dim, entries, block_size, width, dtype, s, 1.0, 1.f, 3);
}

}  // extern "C"
