// extern "C" entry points of the 4-bit pool and of the attention over selected
// blocks (declared in include/minikv.h).  A translation unit of its own, built
// beside abi.cu; argument checks, messages and codes follow abi.cu.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <string>
#include <type_traits>

#include "../../include/minikv.h"
#include "block_select.cuh"
#include "decode_pages.cuh"
#include "int4_pool.cuh"
#include "prefill_int4.cuh"

// in abi.cu's unit
extern "C" int minikv_set_error(int code, const char* message);

namespace {

using namespace minikv;

#define PAGES_REQUIRE(cond, code, msg) \
    do {                               \
        if (!(cond)) return minikv_set_error(code, msg); \
    } while (0)

int cuda_fail(cudaError_t err, const char* where) {
    char text[256];
    std::snprintf(text, sizeof(text), "%s: %s", where, cudaGetErrorString(err));
    return minikv_set_error(MINIKV_ECUDA, text);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool valid_dtype(int d) { return d == MINIKV_F32 || d == MINIKV_F16 || d == MINIKV_BF16; }
bool page_head_dim(int64_t d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

int sm_count() {
    static int cached[64] = {0};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 148;
    if (cached[device] == 0) {
        int n = 0;
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
        cached[device] = n > 0 ? n : 148;
    }
    return cached[device];
}

// Opt-in shared-memory size of a kernel, raised once per device (the limit only grows).
std::mutex g_smem_lock;
template <typename Kernel>
cudaError_t ensure_smem(Kernel kernel, int bytes, int* configured) {
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    const bool tracked = device >= 0 && device < 64;
    std::lock_guard<std::mutex> guard(g_smem_lock);
    if (tracked && configured[device] >= bytes) return cudaSuccess;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err == cudaSuccess && tracked) configured[device] = bytes;
    return err;
}

uint64_t magic_of(int64_t block_size) {  // ceil(2^42 / block_size)
    return ((1ull << 42) + (uint64_t)block_size - 1) / (uint64_t)block_size;
}

// Calls f with integral constants of the head dim.
template <typename F> auto with_dim(int64_t dim, F f) {
    switch (dim) {
        case 32: return f(std::integral_constant<int, 32>());
        case 64: return f(std::integral_constant<int, 64>());
        case 96: return f(std::integral_constant<int, 96>());
        case 128: return f(std::integral_constant<int, 128>());
        case 192: return f(std::integral_constant<int, 192>());
        default: return f(std::integral_constant<int, 256>());
    }
}
template <typename T> struct TypeTag { using type = T; };
template <typename F> auto with_type16(int dtype, F f) {
    return dtype == MINIKV_F16 ? f(TypeTag<__half>()) : f(TypeTag<__nv_bfloat16>());
}
template <typename F> auto with_type(int dtype, F f) {
    return dtype == MINIKV_F32 ? f(TypeTag<float>()) : with_type16(dtype, f);
}

#define POOL_SHAPE_MSG "a 4-bit KV pool needs head_dim 32, 64, 96, 128, 192 or 256"

int check_pool(int64_t num_blocks, int64_t block_size, int64_t kv_heads, int64_t head_dim) {
    PAGES_REQUIRE(num_blocks > 0 && block_size > 0 && kv_heads > 0, MINIKV_EINVAL, "empty batch/heads/cache");
    PAGES_REQUIRE(page_head_dim(head_dim), MINIKV_EINVAL, POOL_SHAPE_MSG);
    PAGES_REQUIRE(block_size <= 1048576 && num_blocks <= 2147483647 / block_size, MINIKV_EINVAL,
                  "KV pool exceeds 2^31 token rows");
    PAGES_REQUIRE(kv_heads <= 65535, MINIKV_EINVAL, "too many KV heads");
    return MINIKV_OK;
}

template <typename Rows>
int run_write(void* kc, void* vc, const void* key, const void* value, int64_t tokens, int64_t num_blocks,
              int64_t block_size, int64_t kv_heads, int64_t head_dim, int64_t k_stride, int64_t v_stride, int dtype,
              Rows map, void* stream) {
    PAGES_REQUIRE(kc && vc && key && value, MINIKV_EINVAL, "null pointer argument");
    PAGES_REQUIRE(aligned16(kc) && aligned16(vc), MINIKV_EINVAL, "KV caches must be 16-byte aligned");
    PAGES_REQUIRE(k_stride >= kv_heads * head_dim && v_stride >= kv_heads * head_dim, MINIKV_EINVAL,
                  "K/V token stride smaller than a row");
    const int64_t es = dtype == MINIKV_F32 ? 4 : 2;
    const bool vec = aligned16(key) && aligned16(value) && k_stride * es % 16 == 0 && v_stride * es % 16 == 0;
    const int sms = sm_count();
    const cudaError_t err = with_type(dtype, [&](auto t) {
        return with_dim(head_dim, [&](auto d) {
            return launch_int4_write<typename decltype(t)::type, decltype(d)::value>(
                kc, vc, key, value, tokens, (int)kv_heads, block_size, k_stride, v_stride, vec, map, sms,
                static_cast<cudaStream_t>(stream));
        });
    });
    if (err != cudaSuccess) return cuda_fail(err, "4-bit KV write launch");
    return MINIKV_OK;
}

// ------------------------------------------------------------------ decode
int check_decode(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks,
                 int64_t block_size, int64_t width, int64_t take, bool selected, int dtype) {
    PAGES_REQUIRE(dtype == MINIKV_F16 || dtype == MINIKV_BF16, MINIKV_EINVAL, "an FP16/BF16 query is required");
    PAGES_REQUIRE(batch > 0 && q_heads > 0, MINIKV_EINVAL, "empty batch/heads/cache");
    const int rc = check_pool(num_blocks, block_size, kv_heads, head_dim);
    if (rc) return rc;
    PAGES_REQUIRE(q_heads % kv_heads == 0, MINIKV_EINVAL, "head dimension or GQA mismatch");
    PAGES_REQUIRE(width > 0, MINIKV_EINVAL, "invalid block table");
    PAGES_REQUIRE(width <= 1048576 / block_size, MINIKV_EINVAL, "maximum table capacity is 1M tokens");
    PAGES_REQUIRE(!selected || (take > 0 && take <= 1048576 / block_size), MINIKV_EINVAL,
                  "selected must list 1 block or more, of 1M tokens at most");
    PAGES_REQUIRE(batch <= 2147483647 / q_heads, MINIKV_EINVAL, "batch/head product too large");
    return MINIKV_OK;
}

// Tiles of 16 tokens: a request's, those of all requests of one head, and a run's are counted in 31 bits.
int check_tiles(int64_t batch, int64_t q_heads, int64_t block_size, int64_t width) {
    const int64_t tiles = width * block_size / 16 + 1;
    PAGES_REQUIRE(tiles <= 2147483647 / batch && tiles <= 2147483647 / q_heads &&
                      batch * tiles <= (1ll << 37) / q_heads,
                  MINIKV_EINVAL, "batch, heads and table capacity together are too large");
    return MINIKV_OK;
}

// Calls f with the consumer type and whether the pool is 4-bit.
template <typename F> auto with_consumer(bool int4, int dtype, int64_t dim, int64_t group, F f) {
    return with_type16(dtype, [&](auto t) {
        return with_dim(dim, [&](auto d) {
            using T = typename decltype(t)::type;
            constexpr int D = decltype(d)::value;
            if (!int4) return f(TypeTag<Wide16Consumer<T, D>>(), t, d, std::false_type());
            return group <= 4 ? f(TypeTag<Int4Consumer<T, D, true>>(), t, d, std::true_type())
                              : f(TypeTag<Int4Consumer<T, D, false>>(), t, d, std::true_type());
        });
    });
}

void decode_plan(bool int4, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int dtype,
                 PageDecodePlan* plan) {
    const int sms = sm_count();
    with_consumer(int4, dtype, dim, q_heads / kv_heads, [&](auto c, auto, auto, auto i) {
        page_decode_plan<typename decltype(c)::type, decltype(i)::value>(batch, q_heads, kv_heads, dim, sms, plan);
        return 0;
    });
}

template <typename T, int D, typename Consumer, bool INT4, bool SELECTED, bool ALIGNED>
cudaError_t launch_page_decode(const PageDecodeParams& p, const PageDecodePlan& plan, cudaStream_t stream) {
    auto kernel = page_decode_kernel<T, D, Consumer, INT4, SELECTED, ALIGNED>;
    static int configured[64] = {0};
    const cudaError_t err = ensure_smem(kernel, plan.smem, configured);
    if (err != cudaSuccess) return err;
    return launch_chained(kernel, dim3((unsigned)plan.grid), dim3(PageShape<Consumer, INT4>::kThreads),
                          (size_t)plan.smem, stream, p);
}

int run_page_decode(bool int4, const void* query, const void* key_cache, const void* value_cache,
                    const int64_t* tables, const int64_t* lens, const int64_t* selected, void* out,
                    unsigned int* tickets, void* workspace, int64_t workspace_bytes, int64_t batch, int64_t q_heads,
                    int64_t kv_heads, int64_t dim, int64_t num_blocks, int64_t block_size, int64_t width,
                    int64_t take, int dtype, void* stream) {
    int rc = check_decode(batch, q_heads, kv_heads, dim, num_blocks, block_size, width, take, selected != nullptr, dtype);
    if (rc == MINIKV_OK) rc = check_tiles(batch, q_heads, block_size, width);
    if (rc) return rc;
    PAGES_REQUIRE(query && key_cache && value_cache && tables && lens && out, MINIKV_EINVAL, "null pointer argument");
    PAGES_REQUIRE(aligned16(query) && aligned16(key_cache) && aligned16(value_cache) && aligned16(out), MINIKV_EINVAL,
                  "query, caches and output must be 16-byte aligned");
    PageDecodePlan plan;
    decode_plan(int4, batch, q_heads, kv_heads, dim, dtype, &plan);
    PAGES_REQUIRE(tickets && workspace && workspace_bytes >= plan.ws_bytes && aligned16(workspace), MINIKV_EINVAL,
                  "decode workspace too small or misaligned");
    PageDecodeParams p{};
    p.q = query;
    p.kc = static_cast<const unsigned char*>(key_cache);
    p.vc = static_cast<const unsigned char*>(value_cache);
    p.tables = tables;
    p.lens = lens;
    p.selected = selected;
    p.out = out;
    p.lse = static_cast<float*>(workspace);
    p.partial = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + plan.ws_lse);
    p.tickets = tickets;
    p.batch = (int)batch;
    p.q_heads = (int)q_heads;
    p.kv_heads = (int)kv_heads;
    p.group = (int)(q_heads / kv_heads);
    p.chunks = plan.chunks;
    p.heads = plan.heads;
    p.num_blocks = (int)num_blocks;
    p.block_size = (int)block_size;
    p.width = (int)width;
    p.take = (int)take;
    p.bs_magic = magic_of(block_size);
    if (int4) {
        p.head_stride = int4_page_bytes(block_size, dim);
        p.row_stride = dim / 2;
        p.page_stride = kv_heads * p.head_stride;
    } else {
        p.head_stride = dim * 2;
        p.row_stride = kv_heads * dim * 2;
        p.page_stride = block_size * p.row_stride;
    }
    p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)dim));
    const cudaError_t err = with_consumer(int4, dtype, dim, q_heads / kv_heads, [&](auto c, auto t, auto d, auto i) {
        using C = typename decltype(c)::type;
        using T = typename decltype(t)::type;
        constexpr int D = decltype(d)::value;
        constexpr bool I = decltype(i)::value;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const bool aligned = block_size % 16 == 0;
        if constexpr (I)
            if (selected == nullptr)
                return aligned ? launch_page_decode<T, D, C, I, false, true>(p, plan, s)
                               : launch_page_decode<T, D, C, I, false, false>(p, plan, s);
        return aligned ? launch_page_decode<T, D, C, I, true, true>(p, plan, s)
                       : launch_page_decode<T, D, C, I, true, false>(p, plan, s);
    });
    if (err != cudaSuccess) return cuda_fail(err, "page decode launch");
    return MINIKV_OK;
}

}  // namespace

extern "C" {

// ------------------------------------------------------------- 4-bit pool
int64_t minikv_int4_page_bytes(int64_t block_size, int64_t head_dim) {
    if (block_size <= 0 || block_size > 1048576 || !page_head_dim(head_dim)) {
        minikv_set_error(MINIKV_EINVAL, POOL_SHAPE_MSG);
        return -1;
    }
    return int4_page_bytes(block_size, head_dim);
}

int minikv_kv_scatter_slots_int4(void* key_cache, void* value_cache, const int64_t* slot_mapping, const void* key,
                                 const void* value, int64_t tokens, int64_t num_blocks, int64_t block_size,
                                 int64_t kv_heads, int64_t head_dim, int64_t key_token_stride,
                                 int64_t value_token_stride, int dtype, void* stream) {
    PAGES_REQUIRE(tokens >= 0, MINIKV_EINVAL, "packed KV slots must be int64 [tokens]");
    PAGES_REQUIRE(valid_dtype(dtype), MINIKV_EINVAL, "packed KV requires FP32/FP16/BF16");
    const int rc = check_pool(num_blocks, block_size, kv_heads, head_dim);
    if (rc) return rc;
    if (tokens == 0) return MINIKV_OK;
    PAGES_REQUIRE(slot_mapping != nullptr, MINIKV_EINVAL, "null pointer argument");
    return run_write(key_cache, value_cache, key, value, tokens, num_blocks, block_size, kv_heads, head_dim,
                     key_token_stride, value_token_stride, dtype, SlotRows{slot_mapping, num_blocks * block_size},
                     stream);
}

int minikv_kv_append_batch_int4(void* key_cache, void* value_cache, const int64_t* block_tables,
                                const int64_t* token_offsets, const void* key, const void* value, int64_t batch,
                                int64_t table_width, int64_t num_blocks, int64_t block_size, int64_t kv_heads,
                                int64_t head_dim, int64_t key_token_stride, int64_t value_token_stride, int dtype,
                                void* stream) {
    PAGES_REQUIRE(batch >= 0 && table_width >= 0, MINIKV_EINVAL, "batch table shape mismatch");
    PAGES_REQUIRE(valid_dtype(dtype), MINIKV_EINVAL, "packed KV requires FP32/FP16/BF16");
    const int rc = check_pool(num_blocks, block_size, kv_heads, head_dim);
    if (rc) return rc;
    if (batch == 0) return MINIKV_OK;
    PAGES_REQUIRE(table_width > 0, MINIKV_EINVAL, "batch table shape mismatch");
    PAGES_REQUIRE(block_tables && token_offsets, MINIKV_EINVAL, "null pointer argument");
    return run_write(key_cache, value_cache, key, value, batch, num_blocks, block_size, kv_heads, head_dim,
                     key_token_stride, value_token_stride, dtype,
                     AppendRows{block_tables, token_offsets, table_width, num_blocks, block_size}, stream);
}

int minikv_kv_gather_slots_int4(const void* key_cache, const void* value_cache, const int64_t* slot_mapping, void* key,
                                void* value, int64_t tokens, int64_t num_blocks, int64_t block_size, int64_t kv_heads,
                                int64_t head_dim, int dtype, void* stream) {
    PAGES_REQUIRE(tokens >= 0, MINIKV_EINVAL, "packed KV slots must be int64 [tokens]");
    PAGES_REQUIRE(valid_dtype(dtype), MINIKV_EINVAL, "packed KV requires FP32/FP16/BF16");
    const int rc = check_pool(num_blocks, block_size, kv_heads, head_dim);
    if (rc) return rc;
    if (tokens == 0) return MINIKV_OK;
    PAGES_REQUIRE(key_cache && value_cache && slot_mapping && key && value, MINIKV_EINVAL, "null pointer argument");
    PAGES_REQUIRE(aligned16(key_cache) && aligned16(value_cache) && aligned16(key) && aligned16(value), MINIKV_EINVAL,
                  "KV caches and outputs must be 16-byte aligned");
    const int sms = sm_count();
    const cudaError_t err = with_type(dtype, [&](auto t) {
        return with_dim(head_dim, [&](auto d) {
            return launch_int4_read<typename decltype(t)::type, decltype(d)::value>(
                key_cache, value_cache, key, value, tokens, (int)kv_heads, block_size,
                SlotRows{slot_mapping, num_blocks * block_size}, sms, static_cast<cudaStream_t>(stream));
        });
    });
    if (err != cudaSuccess) return cuda_fail(err, "minikv_kv_gather_slots_int4 launch");
    return MINIKV_OK;
}

int64_t minikv_paged_decode_int4_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                                 int64_t num_blocks, int64_t block_size, int64_t table_width,
                                                 int dtype) {
    if (check_decode(batch, q_heads, kv_heads, head_dim, num_blocks, block_size, table_width, 1, false, dtype) ||
        check_tiles(batch, q_heads, block_size, table_width))
        return -1;
    PageDecodePlan plan;
    decode_plan(true, batch, q_heads, kv_heads, head_dim, dtype, &plan);
    return plan.ws_bytes;
}

int minikv_paged_decode_int4(const void* query, const void* key_cache, const void* value_cache,
                             const int64_t* block_tables, const int64_t* context_lens, const int64_t* selected,
                             void* out, void* tickets, void* workspace, int64_t workspace_bytes, int64_t batch,
                             int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks,
                             int64_t block_size, int64_t table_width, int64_t max_blocks, int dtype, void* stream) {
    return run_page_decode(true, query, key_cache, value_cache, block_tables, context_lens, selected, out,
                           static_cast<unsigned int*>(tickets), workspace, workspace_bytes, batch, q_heads, kv_heads,
                           head_dim, num_blocks, block_size, table_width, max_blocks, dtype, stream);
}

static int check_prefill(int64_t tokens, int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                         int64_t num_blocks, int64_t block_size, int64_t table_width, int dtype) {
    PAGES_REQUIRE(tokens >= 0 && requests >= 0, MINIKV_EINVAL, "paged prefill metadata shape mismatch");
    const int rc = check_decode(std::max<int64_t>(1, requests), q_heads, kv_heads, head_dim, num_blocks, block_size,
                                table_width, 1, false, dtype);
    if (rc) return rc;
    PAGES_REQUIRE(requests <= 65535, MINIKV_EINVAL, "paged prefill takes up to 65535 requests");
    PAGES_REQUIRE(q_heads / kv_heads <= 64, MINIKV_EUNSUPPORTED, "a 4-bit prefill takes up to 64 query heads a KV head");
    return MINIKV_OK;
}

int64_t minikv_paged_prefill_int4_workspace_bytes(int64_t tokens, int64_t requests, int64_t q_heads, int64_t kv_heads,
                                                  int64_t head_dim, int64_t num_blocks, int64_t block_size,
                                                  int64_t table_width, int dtype) {
    if (check_prefill(tokens, requests, q_heads, kv_heads, head_dim, num_blocks, block_size, table_width, dtype))
        return -1;
    return 0;
}

int minikv_paged_prefill_int4(const void* q, const void* key_cache, const void* value_cache,
                              const int64_t* cu_seqlens_q, const int64_t* query_starts, const int64_t* block_tables,
                              const int64_t* context_lens, void* out, void* /*workspace*/, int64_t /*workspace_bytes*/,
                              int64_t tokens, int64_t requests, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                              int64_t num_blocks, int64_t block_size, int64_t table_width, int64_t max_query_len,
                              int dtype, void* stream) {
    PAGES_REQUIRE(tokens >= 0 && requests >= 0, MINIKV_EINVAL, "paged prefill metadata shape mismatch");
    if (tokens == 0) return MINIKV_OK;
    const int rc = check_prefill(tokens, requests, q_heads, kv_heads, head_dim, num_blocks, block_size, table_width,
                                 dtype);
    if (rc) return rc;
    PAGES_REQUIRE(requests > 0, MINIKV_EINVAL, "paged prefill metadata shape mismatch");
    PAGES_REQUIRE(q && key_cache && value_cache && cu_seqlens_q && query_starts && block_tables && context_lens && out,
                  MINIKV_EINVAL, "null pointer argument");
    PAGES_REQUIRE(aligned16(q) && aligned16(key_cache) && aligned16(value_cache) && aligned16(out), MINIKV_EINVAL,
                  "paged prefill tensors must be 16-byte aligned");
    const int64_t group = q_heads / kv_heads;
    PrefillInt4Params p{};
    p.q = q;
    p.kc = static_cast<const unsigned char*>(key_cache);
    p.vc = static_cast<const unsigned char*>(value_cache);
    p.cu = cu_seqlens_q;
    p.starts = query_starts;
    p.tables = block_tables;
    p.lens = context_lens;
    p.out = out;
    p.tokens = tokens;
    p.width = table_width;
    p.num_blocks = num_blocks;
    p.page_bytes = int4_page_bytes(block_size, head_dim);
    p.requests = (int)requests;
    p.q_heads = (int)q_heads;
    p.kv_heads = (int)kv_heads;
    p.group = (int)group;
    p.block_size = (int)block_size;
    p.tile_tokens = (int)(kPrefillRows / group);
    p.bs_magic = magic_of(block_size);
    p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)head_dim));
    // max_query_len sizes the grid; a longer request's tiles are taken in further turns
    const int64_t longest = std::max<int64_t>(1, std::min(tokens, max_query_len));
    const int64_t tiles = std::min<int64_t>(65535, (longest + p.tile_tokens - 1) / p.tile_tokens);
    const cudaError_t err = with_type16(dtype, [&](auto t) {
        return with_dim(head_dim, [&](auto d) {
            return launch_chained(prefill_int4_kernel<typename decltype(t)::type, decltype(d)::value>,
                                  dim3((unsigned)kv_heads, (unsigned)tiles, (unsigned)requests), dim3(kPrefillThreads),
                                  0, static_cast<cudaStream_t>(stream), p);
        });
    });
    if (err != cudaSuccess) return cuda_fail(err, "minikv_paged_prefill_int4 launch");
    return MINIKV_OK;
}

// --------------------------------------------------------- block selection
int minikv_block_bounds_update(void* bounds, const void* key_cache, const int64_t* block_tables,
                               const int64_t* query_starts, const int64_t* context_lens, int64_t requests,
                               int64_t table_width, int64_t num_blocks, int64_t block_size, int64_t kv_heads,
                               int64_t head_dim, int64_t max_query_len, int pool, void* stream) {
    PAGES_REQUIRE(pool == MINIKV_INT4 || valid_dtype(pool), MINIKV_EINVAL,
                  "key cache must be FP32/FP16/BF16 or a 4-bit pool");
    PAGES_REQUIRE(requests >= 0 && table_width > 0, MINIKV_EINVAL, "block bounds metadata shape mismatch");
    const int rc = check_pool(num_blocks, block_size, kv_heads, head_dim);
    if (rc) return rc;
    PAGES_REQUIRE(table_width <= 1048576 / block_size, MINIKV_EINVAL, "maximum table capacity is 1M tokens");
    if (requests == 0) return MINIKV_OK;
    PAGES_REQUIRE(bounds && key_cache && block_tables && query_starts && context_lens, MINIKV_EINVAL,
                  "null pointer argument");
    PAGES_REQUIRE(aligned16(bounds) && aligned16(key_cache), MINIKV_EINVAL, "caches must be 16-byte aligned");
    // blocks that max_query_len rows can touch
    const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(max_query_len, table_width * block_size));
    const int64_t most = std::min<int64_t>(table_width, (rows + block_size - 2) / block_size + 1);
    const int64_t units = requests * most * kv_heads;
    const int64_t grid = std::min<int64_t>((units + 7) / 8, (int64_t)sm_count() * 8);
    auto run = [&](auto t) {
        return with_dim(head_dim, [&](auto d) {
            return launch_chained(block_bounds_kernel<typename decltype(t)::type, decltype(d)::value>,
                                  dim3((unsigned)grid), dim3(256), 0, static_cast<cudaStream_t>(stream),
                                  static_cast<unsigned char*>(bounds), static_cast<const unsigned char*>(key_cache),
                                  block_tables, query_starts, context_lens, requests, table_width, num_blocks,
                                  (int)block_size, (int)kv_heads, most);
        });
    };
    const cudaError_t err = pool == MINIKV_INT4 ? run(TypeTag<Int4Tag>()) : with_type(pool, run);
    if (err != cudaSuccess) return cuda_fail(err, "minikv_block_bounds_update launch");
    return MINIKV_OK;
}

int minikv_block_bounds_read(const void* bounds, const int64_t* block_ids, int64_t count, float* lower, float* upper,
                             int64_t num_blocks, int64_t kv_heads, int64_t head_dim, void* stream) {
    PAGES_REQUIRE(count >= 0, MINIKV_EINVAL, "block ids must be int64 [count]");
    const int rc = check_pool(num_blocks, 1, kv_heads, head_dim);
    if (rc) return rc;
    if (count == 0) return MINIKV_OK;
    PAGES_REQUIRE(bounds && block_ids && lower && upper, MINIKV_EINVAL, "null pointer argument");
    PAGES_REQUIRE(aligned16(bounds) && aligned16(lower) && aligned16(upper), MINIKV_EINVAL,
                  "bounds and outputs must be 16-byte aligned");
    const int64_t quads = count * kv_heads * (head_dim / 4);
    const int64_t grid = std::min<int64_t>((quads + 255) / 256, (int64_t)sm_count() * 8);
    const cudaError_t err = launch_chained(read_bounds_kernel, dim3((unsigned)grid), dim3(256), 0,
                                           static_cast<cudaStream_t>(stream), static_cast<const unsigned char*>(bounds),
                                           block_ids, count, num_blocks, (int)kv_heads, (int)head_dim,
                                           FastDiv((uint32_t)head_dim / 4), FastDiv((uint32_t)kv_heads), lower, upper);
    if (err != cudaSuccess) return cuda_fail(err, "minikv_block_bounds_read launch");
    return MINIKV_OK;
}

static int check_select(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks,
                        int64_t block_size, int64_t table_width, int64_t max_blocks, int64_t sink, int64_t recent,
                        int dtype) {
    PAGES_REQUIRE(valid_dtype(dtype), MINIKV_EINVAL, "FP32/FP16/BF16 required");
    PAGES_REQUIRE(batch > 0 && q_heads > 0, MINIKV_EINVAL, "empty batch/heads/cache");
    const int rc = check_pool(num_blocks, block_size, kv_heads, head_dim);
    if (rc) return rc;
    PAGES_REQUIRE(q_heads % kv_heads == 0, MINIKV_EINVAL, "head dimension or GQA mismatch");
    PAGES_REQUIRE(table_width > 0 && table_width <= 1048576 / block_size, MINIKV_EINVAL,
                  "maximum table capacity is 1M tokens");
    PAGES_REQUIRE(max_blocks > 0 && max_blocks <= 1048576 && sink >= 0 && recent >= 0 &&
                      sink + recent <= max_blocks,
                  MINIKV_EINVAL, "max_blocks must be positive and hold the sink and recent blocks");
    PAGES_REQUIRE(batch <= 2147483647 / std::max<int64_t>(kv_heads, table_width), MINIKV_EINVAL, "batch/head product too large");
    return MINIKV_OK;
}

int64_t minikv_select_blocks_workspace_bytes(int64_t batch, int64_t kv_heads, int64_t table_width) {
    if (batch <= 0 || kv_heads <= 0 || table_width <= 0) return -1;
    return batch * kv_heads * table_width * 4;
}

int minikv_select_blocks(const void* query, const void* bounds, const int64_t* block_tables,
                         const int64_t* context_lens, int64_t* selected, void* workspace, int64_t workspace_bytes,
                         int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks,
                         int64_t block_size, int64_t table_width, int64_t max_blocks, int64_t sink_blocks,
                         int64_t recent_blocks, int dtype, void* stream) {
    const int rc = check_select(batch, q_heads, kv_heads, head_dim, num_blocks, block_size, table_width, max_blocks,
                                sink_blocks, recent_blocks, dtype);
    if (rc) return rc;
    PAGES_REQUIRE(query && bounds && block_tables && context_lens && selected && workspace, MINIKV_EINVAL,
                  "null pointer argument");
    PAGES_REQUIRE(aligned16(bounds), MINIKV_EINVAL, "bounds must be 16-byte aligned");
    PAGES_REQUIRE(workspace_bytes >= minikv_select_blocks_workspace_bytes(batch, kv_heads, table_width), MINIKV_EINVAL,
                  "select_blocks workspace too small");
    SelectParams p{};
    p.q = query;
    p.bounds = static_cast<const unsigned char*>(bounds);
    p.tables = block_tables;
    p.lens = context_lens;
    p.keys = static_cast<uint32_t*>(workspace);
    p.selected = selected;
    p.width = table_width;
    p.num_blocks = num_blocks;
    p.q_heads = (int)q_heads;
    p.kv_heads = (int)kv_heads;
    p.group = (int)(q_heads / kv_heads);
    p.block_size = (int)block_size;
    p.take = (int)max_blocks;
    p.sink = (int)sink_blocks;
    p.recent = (int)recent_blocks;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t err = cudaSuccess;
    if (table_width > max_blocks) {  // else every request takes all of its blocks
        const int64_t head_groups = (kv_heads + kScoreHeads - 1) / kScoreHeads;
        // as many spans as two CTAs a SM (one from 192 dims) hold at once, each of whole turns of 8 warps
        const int64_t spans = std::max<int64_t>(1, (head_dim <= 128 ? 2 : 1) * sm_count() / (batch * head_groups));
        const int64_t span = std::min<int64_t>(kScoreSpan, ((table_width + spans - 1) / spans + 7) / 8 * 8);
        p.span = (int)span;
        const dim3 grid((unsigned)(batch * ((table_width + span - 1) / span)), (unsigned)head_groups);
        err = with_type(dtype, [&](auto t) {
            return with_dim(head_dim, [&](auto d) {
                using T = typename decltype(t)::type;
                constexpr int D = decltype(d)::value;
                return launch_chained(kv_heads % kScoreHeads == 0 ? score_blocks_kernel<T, D, true>
                                                                  : score_blocks_kernel<T, D, false>,
                                      grid, dim3(256), 0, s, p);
            });
        });
        if (err != cudaSuccess) return cuda_fail(err, "minikv_select_blocks scores");
    }
    if (table_width <= 4096) {
        const int keys = table_width <= 512 ? 1 : table_width <= 1024 ? 2 : table_width <= 2048 ? 4 : 8;
        const int threads = (int)(((table_width + keys - 1) / keys + 31) / 32 * 32);
        const dim3 grid((unsigned)(batch * kv_heads));
        err = keys == 1   ? launch_chained(select_few_kernel<1>, grid, dim3(threads), 0, s, p)
              : keys == 2 ? launch_chained(select_few_kernel<2>, grid, dim3(threads), 0, s, p)
              : keys == 4 ? launch_chained(select_few_kernel<4>, grid, dim3(threads), 0, s, p)
                          : launch_chained(select_few_kernel<8>, grid, dim3(threads), 0, s, p);
        if (err != cudaSuccess) return cuda_fail(err, "minikv_select_blocks launch");
        return MINIKV_OK;
    }
    const int held = (int)std::min<int64_t>(table_width, kSelectHeld);
    static int configured[64] = {0};
    err = ensure_smem(select_blocks_kernel, kSelectHeld * 4, configured);
    if (err == cudaSuccess)
        err = launch_chained(select_blocks_kernel, dim3((unsigned)(batch * kv_heads)), dim3(kSelectThreads),
                             (size_t)held * 4, s, p, held);
    if (err != cudaSuccess) return cuda_fail(err, "minikv_select_blocks launch");
    return MINIKV_OK;
}

int64_t minikv_paged_decode_selected_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                     int64_t head_dim, int64_t num_blocks, int64_t block_size,
                                                     int64_t table_width, int dtype) {
    if (check_decode(batch, q_heads, kv_heads, head_dim, num_blocks, block_size, table_width, 1, false, dtype) ||
        check_tiles(batch, q_heads, block_size, table_width))
        return -1;
    PageDecodePlan plan;
    decode_plan(false, batch, q_heads, kv_heads, head_dim, dtype, &plan);
    return plan.ws_bytes;
}

int minikv_paged_decode_selected(const void* query, const void* key_cache, const void* value_cache,
                                 const int64_t* block_tables, const int64_t* context_lens, const int64_t* selected,
                                 void* out, void* tickets, void* workspace, int64_t workspace_bytes, int64_t batch,
                                 int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks,
                                 int64_t block_size, int64_t table_width, int64_t max_blocks, int dtype,
                                 void* stream) {
    PAGES_REQUIRE(selected != nullptr, MINIKV_EINVAL, "null pointer argument");
    return run_page_decode(false, query, key_cache, value_cache, block_tables, context_lens, selected, out,
                           static_cast<unsigned int*>(tickets), workspace, workspace_bytes, batch, q_heads, kv_heads,
                           head_dim, num_blocks, block_size, table_width, max_blocks, dtype, stream);
}

}  // extern "C"
