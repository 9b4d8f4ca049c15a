// The ways to compute an attention: on tiles (attention_tiles.hip), for few queries along split keys (attention_few.hip), and a row at a time
// (attention.hip).
#pragma once

#include "attention_device.h"

namespace mg {

// What a float16 result leaves out is kept as this times it, in float16: 2^11, so that it is about as large as the result.
constexpr float kRest = 2048.0f;

// In float16 the last piece of a row in LDS may hold values of the next one, which meet zeros: scores that come out as no number need not be.
__device__ __forceinline__ bool shares_pieces(const Attention &p, int size) { return p.D * size % 16 != 0; }

bool tiles_take(const Attention &p, int size, uintptr_t ends);
int forward_tiles(const Attention &p, int dtype, const void *q, const void *k, const void *v, void *out, void *rest, void *lse);

// Whether the forward pass and dq go 32 columns a block instead of 128 queries.
bool few_take(const Attention &p, int size);
int forward_few(const Attention &p, int dtype, const void *q, const void *k, const void *v, void *out, void *rest, void *lse);

struct Stats;
size_t few_dq_bytes(const Attention &p);  // of workspace for dq_few
int dq_few(const Attention &p, const Stats &stats, int dtype, const void *q, const void *k, const void *v, const void *grad, const void *lse, void *dq,
           float *sums);
int backward_tiles(const Attention &p, int dtype, const void *q, const void *k, const void *v, const void *out, const void *rest, const void *lse,
                   const void *grad, void *dq, void *dk, void *dv);

}  // namespace mg
