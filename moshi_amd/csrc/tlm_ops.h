// Launches of the operators that stand by themselves behind the C ABI and inside a token LM's step (tlm_ops.hip).
#pragma once
#include "tlm_kv8.h"

// dtype of keys, values and queries: MMI_BF16 or MMI_F32 (a.k / a.v / a.x); f32: fp32 results, from operands of two parts (fp32 queries; otherwise bf16 from one)
int tlm_kv8_append(hipStream_t s, TlmKv8Append a, int dtype);
// fills in how the work is split (`cap`: pages that a sequence can have at most; `room`: floats that a workspace may have) and says what workspace
// that takes, in floats
size_t tlm_kv8_plan(TlmKv8Attn& a, long cap, size_t room);
void tlm_kv8_workspace(TlmKv8Attn& a, float* workspace);      // aligned to 16 bytes
int tlm_kv8_attend(hipStream_t s, const TlmKv8Attn& a, int dtype, bool f32);

// rows of several tensors; row r of a group of `beams` becomes a copy of what row parent[r] of it was (row: where the groups' rows are, null: in order)
constexpr int BEAM_MAX = 32;
struct TlmReorderTensor { void* p; int64_t stride, bytes; };
int tlm_reorder(hipStream_t s, int n, const TlmReorderTensor* tensors, int groups, int beams, const int* parent, const int* row);
