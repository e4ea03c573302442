// gsd_internal.h — launchers of the decoder's kernels (called by gsd_capi.cpp).
#pragma once

#include <hip/hip_runtime.h>

#include "../../../include/gsrdecoder.h"

namespace gsd {

// MI355X: 256 compute units in 8 dies, each with its own L2.
constexpr int kComputeUnits = 256;
constexpr int64_t kLastCacheBytes = INT64_C(256) << 20;  // of the one that all dies share

hipError_t launch_rotary(const gsd_rotary& a, hipStream_t st);

hipError_t launch_rms_norm(const gsd_norm& a, void* y, uint8_t* y8, float* scale, hipStream_t st);
// rows of partial sums of dweight
int64_t norm_backward_groups(int64_t rows, int64_t width);
hipError_t launch_rms_norm_backward(int dtype, int64_t rows, int64_t width, const void* h,
                                    const float* rstd, const void* weight, const void* dy,
                                    int64_t dy_stride, const void* dh, int64_t dh_stride,
                                    void* dx, void* dweight, float* partial, hipStream_t st);

// How an attention pass is split: `parts` shares of the long axis per block of
// the short one, joined by a second kernel when there is more than one.
struct AttentionSplit {
    int64_t blocks;  // blocks of rows (forward, dq) or of keys (dk, dv), per batch and kv head
    int64_t tiles;   // tiles of the axis that is walked
    int64_t parts;
};
AttentionSplit attention_split_rows(const gsd_attention& a);      // forward
AttentionSplit attention_split_dq(const gsd_attention& a);
AttentionSplit attention_split_dkdv(const gsd_attention& a);

// partial_o [parts, batch kv_heads, rows, dim], partial_lse [parts, batch kv_heads, rows];
// list [batch (keys + 1)] where there is a mask, else null
hipError_t launch_attention(const gsd_attention& a, const AttentionSplit& sp, float* partial_o,
                            float* partial_lse, int32_t* list, hipStream_t st);

struct AttentionBackwardBuffers {
    float* stat;         // [batch kv_heads, 2, rows]
    // (fp16) the largest |do| and |delta| per block of rows, [batch kv_heads, 2, top_blocks],
    // and |v| per block of keys, [batch kv_heads, value_blocks]
    float* top;
    float* value_top;
    float* partial_dq;   // [parts, batch kv_heads, rows, dim]
    float* partial_dk;   // [parts, batch kv_heads, keys, dim]
    float* partial_dv;
    int32_t* list;       // [batch (keys + 1)] where there is a mask
};
int64_t attention_top_blocks(const gsd_attention& a);
int64_t attention_value_blocks(const gsd_attention& a);
hipError_t launch_attention_backward(const gsd_attention& a, const gsd_attention_grad& g,
                                     const AttentionSplit& sq, const AttentionSplit& sk,
                                     const AttentionBackwardBuffers& buf, hipStream_t st);

}  // namespace gsd
