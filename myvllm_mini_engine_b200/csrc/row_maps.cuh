// Where the KV writes put a token's row (16-bit, fp8 and 4-bit pools).
#pragma once

#include <stdint.h>

namespace minikv {

// Row destination for the three write forms.  Returns -1 for "skip".
struct SlotRows {         // data.cu:196-206
    const int64_t* slots;
    int64_t capacity;
    __device__ int64_t operator()(int64_t t) const {
        const int64_t s = slots[t];
        return (s >= 0 && s < capacity) ? s : -1;
    }
};
struct AppendRows {       // data.cu:89-107
    const int64_t* tables; const int64_t* offsets;
    int64_t width, num_blocks, block_size;
    __device__ int64_t operator()(int64_t r) const {
        const int64_t logical = offsets[r];
        if (logical < 0) return -1;
        const int64_t index = logical / block_size;
        if (index >= width) return -1;
        const int64_t page = tables[r * width + index];
        if (page < 0 || page >= num_blocks) return -1;
        return page * block_size + logical % block_size;
    }
};
struct RangeRows {        // data.cu:68-86
    const int64_t* ids; int64_t num_ids, offset, num_blocks, block_size;
    __device__ int64_t operator()(int64_t t) const {
        const int64_t logical = offset + t;
        const int64_t index = logical / block_size;
        if (logical < 0 || index >= num_ids) return -1;
        const int64_t page = ids[index];
        if (page < 0 || page >= num_blocks) return -1;
        return page * block_size + logical % block_size;
    }
};

}  // namespace minikv
