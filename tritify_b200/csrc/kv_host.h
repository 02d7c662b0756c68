// The KV cache's entry points without their locking, for callers that hold the context's lock (the attention half of a
// decoder block, ktmoe.cu). Arguments as in include/ktmoe.h.
#pragma once

#include "ktmoe.h"

int kv_append(ktmoe_ctx* ctx, const ktmoe_kv_cache* cache, const ktmoe_kv_batch* batch, const int32_t* k, int64_t ld_k,
              const int32_t* v, int64_t ld_v, const ktmoe_scale* k_scale, const ktmoe_scale* v_scale,
              int32_t scale_stride, const ktmoe_rope* rope, void* stream);
int kv_attention(ktmoe_ctx* ctx, const ktmoe_kv_cache* cache, const ktmoe_kv_batch* batch, const int32_t* q, int64_t ld_q,
                 const ktmoe_scale* scale, int32_t scale_stride, const ktmoe_rope* rope, int32_t n_heads,
                 double softmax_scale, int32_t window, int32_t sinks, int32_t* o, int64_t ld_o, ktmoe_scale* o_scale,
                 void* stream);
