// attn.hip — attention over the quantised cache (include/hako_attn.h): single
// tokens of many sequences, and whole packed prompts.
#include "kv.h"

namespace hako {
namespace {

constexpr int kMaxGroup = 16;    // query heads per key/value head
constexpr int kSeqs = 128;       // sequences of one prompt launch (by value in the kernel arguments)

struct AttnKv {
	const uint8_t *k, *v;
	const float *ks, *vs;
	int n_slots, max_seq, kvh;
	int prefix_slot, prefix_len;
};

struct SeqTab {
	int n;
	int row[kSeqs + 1], slot[kSeqs], start[kSeqs];
};

template <bool Q8>
__device__ __forceinline__ float code(const uint8_t *p, size_t i) {
	return Q8 ? (float)((const int8_t *)p)[i] : (float)((const _Float16 *)p)[i];
}

// One wave per query row and head: positions one after the other, a running
// maximum and sum.
template <int HD, bool Q8>
__device__ __forceinline__ void attend(const AttnKv &c, int slot, int end, const float *q, float *out, int kvh,
                                       float scale) {
	constexpr int N = HD / 64;
	const int lane = threadIdx.x;
	float qv[N], o[N];
#pragma unroll
	for (int i = 0; i < N; i++) {
		qv[i] = q[lane + 64 * i] * scale;
		o[i] = 0.0f;
	}
	float m = -INFINITY, l = 0.0f;
	for (int p = 0; p < end; p++) {
		const size_t r = ((size_t)(p < c.prefix_len ? c.prefix_slot : slot) * c.kvh + kvh) * c.max_seq + p;
		float s = 0.0f;
#pragma unroll
		for (int i = 0; i < N; i++) s = __builtin_fmaf(qv[i], code<Q8>(c.k, r * HD + lane + 64 * i), s);
		s = wave_sum(s) * c.ks[r];
		const float mn = s > m ? s : m;
		const float a = m == -INFINITY ? 0.0f : expf(m - mn);
		const float w = expf(s - mn), wv = w * c.vs[r];
		l = l * a + w;
#pragma unroll
		for (int i = 0; i < N; i++) o[i] = __builtin_fmaf(wv, code<Q8>(c.v, r * HD + lane + 64 * i), o[i] * a);
		m = mn;
	}
#pragma unroll
	for (int i = 0; i < N; i++) out[lane + 64 * i] = end > 0 ? o[i] / l : 0.0f;
}

template <int HD, bool Q8>
__global__ __launch_bounds__(64) void decode_kernel(AttnKv c, float *out, int64_t ldo, const float *q, int64_t ldq,
                                                    const int *__restrict__ slot, const int *__restrict__ len, int G,
                                                    float scale) {
	const int s = blockIdx.x, h = blockIdx.y;
	const int sl = slot ? slot[s] : s;
	int end = min(max(len[s], 0), c.max_seq);
	if (sl < 0 || sl >= c.n_slots) end = 0;
	attend<HD, Q8>(c, sl, end, q + s * ldq + h * HD, out + s * ldo + h * HD, h / G, scale);
}

template <int HD, bool Q8>
__global__ __launch_bounds__(64) void prompt_kernel(AttnKv c, SeqTab t, float *out, int64_t ldo, const float *q,
                                                    int64_t ldq, int G, float scale) {
	const int row = blockIdx.x, h = blockIdx.y;
	int s = 0;
	while (row >= t.row[s + 1]) s++;
	attend<HD, Q8>(c, t.slot[s], t.start[s] + row - t.row[s] + 1, q + row * ldq + h * HD, out + row * ldo + h * HD,
	               h / G, scale);
}

int attn_check(float *out, int64_t ldo, const float *q, int64_t ldq, const hako_gpu_kv *kv, int n_seq, int H,
               int prefix_slot, int prefix_len) {
	if (int rc = kv_check(kv)) return rc;
	if (n_seq < 0) return set_error(HAKO_GPU_EINVAL, "%d sequences", n_seq);
	if (H < 1 || H > 65535 || H % kv->n_kv_heads || H / kv->n_kv_heads > kMaxGroup)
		return set_error(HAKO_GPU_EINVAL, "%d query heads over %d key/value heads (at most %d to one)", H,
		                 kv->n_kv_heads, kMaxGroup);
	if (int rc = rows_check("q", q, ldq, (int64_t)H * kv->head_dim)) return rc;
	if (int rc = rows_check("out", out, ldo, (int64_t)H * kv->head_dim)) return rc;
	if (q == out && ldq != ldo) return set_error(HAKO_GPU_EINVAL, "attention in place with two strides");
	if (prefix_len < 0 || prefix_len > kv->max_seq ||
	    (prefix_len > 0 && (prefix_slot < 0 || prefix_slot >= kv->n_slots)))
		return set_error(HAKO_GPU_EINVAL, "prefix of %d positions in slot %d: %d slots of %d positions", prefix_len,
		                 prefix_slot, kv->n_slots, kv->max_seq);
	return HAKO_GPU_OK;
}

AttnKv attn_kv(const hako_gpu_kv *kv, int prefix_slot, int prefix_len) {
	return {(const uint8_t *)kv->k, (const uint8_t *)kv->v, kv->k_scale, kv->v_scale, kv->n_slots, kv->max_seq,
	        kv->n_kv_heads, prefix_slot, prefix_len};
}

}  // namespace
}  // namespace hako

using namespace hako;

#define HK_KV_SWITCH(kv, CALL)                             \
	do {                                                   \
		if ((kv)->head_dim == 128) {                       \
			if ((kv)->type == HAKO_KV_Q8) CALL(128, true); \
			else CALL(128, false);                         \
		} else {                                           \
			if ((kv)->type == HAKO_KV_Q8) CALL(64, true);  \
			else CALL(64, false);                          \
		}                                                  \
	} while (0)

extern "C" {

int hako_gpu_attn_decode(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                         const int *slot, const int *len, int n_seq, int n_heads, float scale, int prefix_slot,
                         int prefix_len) {
	if (int rc = attn_check(out, out_stride, q, q_stride, kv, n_seq, n_heads, prefix_slot, prefix_len)) return rc;
	if (!len && n_seq) return set_error(HAKO_GPU_EINVAL, "null lengths");
	if (!slot && n_seq > kv->n_slots)
		return set_error(HAKO_GPU_EINVAL, "%d sequences without slots in a cache of %d", n_seq, kv->n_slots);
	if (int rc = require_device()) return rc;
	if (n_seq == 0) return ok();
	const AttnKv c = attn_kv(kv, prefix_slot, prefix_len);
#define HK_DECODE(HD, Q8)                                                                                          \
	hipLaunchKernelGGL((decode_kernel<HD, Q8>), dim3(n_seq, n_heads), dim3(64), 0, stream(), c, out, out_stride, q, \
	                   q_stride, slot, len, n_heads / kv->n_kv_heads, scale)
	HK_KV_SWITCH(kv, HK_DECODE);
#undef HK_DECODE
	HK_LAUNCHED("attention");
	return ok();
}

int hako_gpu_attn_prompt(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                         const int *slot, const int *start, const int *len, int n_seq, int n_heads, float scale,
                         int prefix_slot, int prefix_len) {
	if (int rc = attn_check(out, out_stride, q, q_stride, kv, n_seq, n_heads, prefix_slot, prefix_len)) return rc;
	if (n_seq && (!start || !len)) return set_error(HAKO_GPU_EINVAL, "null starts or lengths");
	int64_t rows = 0;
	for (int s = 0; s < n_seq; s++) {
		const int sl = slot ? slot[s] : s;
		if (sl < 0 || sl >= kv->n_slots) return set_error(HAKO_GPU_EINVAL, "sequence %d in slot %d of %d", s, sl, kv->n_slots);
		if (start[s] < 0 || len[s] < 0 || start[s] > kv->max_seq || len[s] > kv->max_seq - start[s])
			return set_error(HAKO_GPU_EINVAL, "sequence %d: %d tokens from position %d in %d positions", s, len[s],
			                 start[s], kv->max_seq);
		rows += len[s];
	}
	if (rows > 0x7FFFFFFF) return set_error(HAKO_GPU_EINVAL, "%lld tokens in one call", (long long)rows);
	if (int rc = require_device()) return rc;
	const AttnKv c = attn_kv(kv, prefix_slot, prefix_len);
	int64_t row = 0;
	for (int s = 0; s < n_seq;) {
		SeqTab t;
		t.n = 0;
		t.row[0] = 0;
		const int64_t row0 = row;
		for (; s < n_seq && t.n < kSeqs; s++) {
			if (len[s] == 0) continue;
			t.slot[t.n] = slot ? slot[s] : s;
			t.start[t.n] = start[s];
			row += len[s];
			t.row[++t.n] = (int)(row - row0);
		}
		if (t.n == 0) break;
#define HK_PROMPT(HD, Q8)                                                                                          \
	hipLaunchKernelGGL((prompt_kernel<HD, Q8>), dim3((unsigned)(row - row0), n_heads), dim3(64), 0, stream(), c, t, \
	                   out + row0 * out_stride, out_stride, q + row0 * q_stride, q_stride, n_heads / kv->n_kv_heads, scale)
		HK_KV_SWITCH(kv, HK_PROMPT);
#undef HK_PROMPT
		HK_LAUNCHED("attention");
	}
	return ok();
}

}  // extern "C"
