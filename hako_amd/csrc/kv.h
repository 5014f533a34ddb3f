// kv.h — the quantised cache as the kernels see it (include/hako_attn.h).
#pragma once
#include "../../include/hako_attn.h"
#include "hako_dev.h"
#include "hako_rt.h"

namespace hako {

// Threads of a launch's grid that HIP takes.
constexpr int64_t kMaxThreads = 0xFFFFFFFFll;
// Bytes of a code.
inline int kv_elt(int type) { return type == HAKO_KV_Q8 ? 1 : 2; }
// The checks every call makes of its cache; 0 or an error code.
int kv_check(const hako_gpu_kv *kv);
// ... and of a row pointer and stride (floats): 16-byte rows of at least `width`.
int rows_check(const char *what, const void *p, int64_t stride, int64_t width);

// hako_gpu_attn_decode without its checks, over len[i] + len_add positions;
// n_seq >= 1.
int attn_decode(float *out, int64_t ldo, const float *q, int64_t ldq, const hako_gpu_kv *kv, const int *slot,
                const int *len, int len_add, int n_seq, int H, float scale, int prefix_slot, int prefix_len);
// The workspace of such calls, taken now (before a capture).
int attn_decode_reserve(const hako_gpu_kv *kv, int n_seq, int H, int prefix_len);

}  // namespace hako
