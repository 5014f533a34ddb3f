// kvcache.hip — the quantised key/value cache: tokens appended (their queries
// and keys rotated in the same pass) and rows read back.
#include "kv.h"

namespace hako {

// A cache's type and shape; 0 or an error code.
static int kv_shape_check(const hako_gpu_kv *kv) {
	if (!kv) return set_error(HAKO_GPU_EINVAL, "null cache");
	if (kv->type != HAKO_KV_F16 && kv->type != HAKO_KV_Q8)
		return set_error(HAKO_GPU_ETYPE, "cache type %d", kv->type);
	if (kv->n_slots < 1 || kv->max_seq < 1 || kv->n_kv_heads < 1 || kv->n_kv_heads > 65535 ||
	    (kv->head_dim != 64 && kv->head_dim != 128))
		return set_error(HAKO_GPU_EINVAL, "unsupported cache shape: %d slots of %d positions, %d heads of %d",
		                 kv->n_slots, kv->max_seq, kv->n_kv_heads, kv->head_dim);
	// one slot and head is read through 32-bit buffer offsets
	if ((size_t)kv->max_seq * kv->head_dim * kv_elt(kv->type) >= kBufNone)
		return set_error(HAKO_GPU_EINVAL, "max_seq %d x head_dim %d: one head's rows exceed 2 GiB", kv->max_seq,
		                 kv->head_dim);
	// at most 2^48 - 1 rows, so that no size in bytes overflows (a slot's rows, 25 bits by 16, do not; all slots' might)
	const uint64_t slot_rows = (uint64_t)kv->max_seq * kv->n_kv_heads;
	if ((uint64_t)kv->n_slots > ((1ull << 48) - 1) / slot_rows)
		return set_error(HAKO_GPU_EINVAL, "%d slots of %d positions of %d heads", kv->n_slots, kv->max_seq, kv->n_kv_heads);
	return HAKO_GPU_OK;
}

int kv_check(const hako_gpu_kv *kv) {
	if (int rc = kv_shape_check(kv)) return rc;
	if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale) return set_error(HAKO_GPU_EINVAL, "null cache array");
	if ((((uintptr_t)kv->k | (uintptr_t)kv->v) & 15) || (((uintptr_t)kv->k_scale | (uintptr_t)kv->v_scale) & 3))
		return set_error(HAKO_GPU_EINVAL, "cache arrays need 16-byte (codes) and 4-byte (scales) alignment");
	return HAKO_GPU_OK;
}

int rows_check(const char *what, const void *p, int64_t stride, int64_t width) {
	if (!p) return set_error(HAKO_GPU_EINVAL, "null %s", what);
	if ((uintptr_t)p & 15) return set_error(HAKO_GPU_EINVAL, "%s is not 16-byte aligned", what);
	if (stride < width || (stride & 3))
		return set_error(HAKO_GPU_EINVAL, "%s stride %lld: a multiple of 4 of at least %lld floats is wanted", what,
		                 (long long)stride, (long long)width);
	return HAKO_GPU_OK;
}

namespace {

struct KvDev {
	uint8_t *k, *v;
	float *ks, *vs;
	int n_slots, max_seq, kvh;
};

KvDev kv_dev(const hako_gpu_kv *kv) {
	return {(uint8_t *)kv->k, (uint8_t *)kv->v, kv->k_scale, kv->v_scale, kv->n_slots, kv->max_seq, kv->n_kv_heads};
}

struct RopeDev {
	const float *table;
	int n_pos, rot, interleaved;
};

// Largest of the L lanes (8 or 16) of a row, as unsigned bits.
template <int L>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
	v = max(v, (uint32_t)dpp_i<kDppQuadSwap1>((int)v));
	v = max(v, (uint32_t)dpp_i<kDppQuadSwap2>((int)v));
	v = max(v, (uint32_t)dpp_i<kDppHalfMirror>((int)v));
	if (L == 16) v = max(v, (uint32_t)dpp_i<kDppMirror>((int)v));
	return v;
}

// a*c - b*s and a*s + b*c, each product and sum rounded (no fused form): the
// codes of a key then follow from its definition alone.
__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
#pragma clang fp contract(off)
	const float ac = a * c, bs = b * s, as = a * s, bc = b * c;
	a = ac - bs;
	b = as + bc;
}

// One lane's 8 values of a head row as codes at dims 4*u0.. and 4*u1.. of
// `codes`, and (one lane) the row's scale.
template <int L, bool Q8>
__device__ __forceinline__ void put_row(const float v[8], int u0, int u1, uint8_t *codes, float *scale, bool first) {
	uint32_t m = 0;
#pragma unroll
	for (int i = 0; i < 8; i++) m = max(m, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
	m = row_max<L>(m);
	const bool finite = m < 0x7F800000u;
	float sc;
	if (Q8) {
		const float amax = m < 0x00800000u ? 0.0f : __builtin_bit_cast(float, m);
		sc = q8_xs(amax);
		const float inv = finite ? q8_inv(amax, sc) : 0.0f;
		uint32_t w[2];
#pragma unroll
		for (int h = 0; h < 2; h++) {
			w[h] = 0;
#pragma unroll
			for (int i = 0; i < 4; i++) w[h] |= q8_code(ftz(v[4 * h + i]), inv) << (8 * i);
		}
		*(uint32_t *)(codes + 4 * u0) = w[0];
		*(uint32_t *)(codes + 4 * u1) = w[1];
	} else {
		const int e = finite ? max((int)(m >> 23) - 127, -126) : 0;
		sc = __builtin_ldexpf(1.0f, e);
		uint2 w[2];
#pragma unroll
		for (int h = 0; h < 2; h++) {
			uint16_t c[4];
#pragma unroll
			for (int i = 0; i < 4; i++)
				c[i] = finite ? __builtin_bit_cast(uint16_t, (_Float16)__builtin_ldexpf(v[4 * h + i], -e)) : 0;
			w[h] = make_uint2(c[0] | ((uint32_t)c[1] << 16), c[2] | ((uint32_t)c[3] << 16));
		}
		*(uint2 *)(codes + 8 * u0) = w[0];
		*(uint2 *)(codes + 8 * u1) = w[1];
	}
	if (first) *scale = finite ? sc : __builtin_nanf("");
}

// Four floats past the caches: for long runs of values that fill none of them
// usefully (reading 32.7 thousand positions of 4 heads back: 26 us, 44 with
// ordinary stores).
__device__ __forceinline__ void put4_past(float *dst, const float x[4]) {
	typedef float f4 __attribute__((ext_vector_type(4)));
	__builtin_nontemporal_store((f4){x[0], x[1], x[2], x[3]}, (f4 *)dst);
}

// A head row (token, one of its query, key or value heads) is L = head_dim/8
// lanes of two float4 each. The two of a lane hold whole pairs: unit u (dims
// 4u..4u+3) with unit u + rot/8 in the half layout, any two in the
// interleaved one. Lanes on consecutive units keep both accesses contiguous;
// a row's maximum is three or four lane permutes, nothing passes through LDS.
//
// Bound: memory, and below some thousand rows the launch (one token 3 us, 512
// of 7B heads 5.7). 8192 packed tokens of 7B heads into 16 bits move 286 MB in
// 51 us, 5.6 TB/s (a copy of 1 GiB runs at 5.1; part of the input is still in
// the caches), the waves waiting 79% of their cycles.
template <int HD, bool Q8>
__global__ __launch_bounds__(256) void append_kernel(KvDev kv, const int *__restrict__ slot, const int *__restrict__ posv,
                                                     int n_tok, const float *__restrict__ k,
                                                     const float *__restrict__ v, int64_t kv_stride, RopeDev rope,
                                                     const float *q, float *q_out, int H, int64_t q_stride,
                                                     int64_t q_out_stride) {
	constexpr int L = HD / 8;
	const uint32_t row = blockIdx.x * (256 / L) + threadIdx.x / L, per = H + 2 * kv.kvh;
	const int tok = (int)(row / per), h = (int)(row - tok * per), t = threadIdx.x % L;
	if (tok >= n_tok) return;
	const int sl = slot ? slot[tok] : tok, pos = posv[tok];
	if (sl < 0 || sl >= kv.n_slots || pos < 0 || pos >= kv.max_seq || (rope.table && pos >= rope.n_pos)) return;
	const bool is_q = h < H, is_v = h >= H + kv.kvh;
	const float *src = is_q ? q + tok * q_stride + (int64_t)h * HD
	                        : (is_v ? v + tok * kv_stride + (int64_t)(h - H - kv.kvh) * HD
	                                : k + tok * kv_stride + (int64_t)(h - H) * HD);
	const int ru = rope.table && !is_v ? rope.rot / 8 : 0;   // rotated units: 2 ru
	const int u0 = t < ru ? t : t + ru, u1 = t < ru ? t + ru : t + L;
	const float4 a = *(const float4 *)(src + 4 * u0), b = *(const float4 *)(src + 4 * u1);
	float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
	if (t < ru) {
		const float *tb = rope.table + (size_t)pos * rope.rot;
		if (rope.interleaved) {
			const float4 c0 = *(const float4 *)(tb + 4 * u0), c1 = *(const float4 *)(tb + 4 * u1);
			turn(x[0], x[1], c0.x, c0.y);
			turn(x[2], x[3], c0.z, c0.w);
			turn(x[4], x[5], c1.x, c1.y);
			turn(x[6], x[7], c1.z, c1.w);
		} else {
			const float4 c0 = *(const float4 *)(tb + 8 * t), c1 = *(const float4 *)(tb + 8 * t + 4);
			turn(x[0], x[4], c0.x, c0.y);
			turn(x[1], x[5], c0.z, c0.w);
			turn(x[2], x[6], c1.x, c1.y);
			turn(x[3], x[7], c1.z, c1.w);
		}
	}
	if (is_q) {
		float *dst = q_out + tok * q_out_stride + (int64_t)h * HD;
		*(float4 *)(dst + 4 * u0) = make_float4(x[0], x[1], x[2], x[3]);
		*(float4 *)(dst + 4 * u1) = make_float4(x[4], x[5], x[6], x[7]);
		return;
	}
	const int hh = is_v ? h - H - kv.kvh : h - H;
	const size_t r = ((size_t)sl * kv.kvh + hh) * kv.max_seq + pos;
	put_row<L, Q8>(x, u0, u1, (is_v ? kv.v : kv.k) + r * HD * (Q8 ? 1 : 2), (is_v ? kv.vs : kv.ks) + r, t == 0);
}

// A thread takes four consecutive dims of kReadRows rows, loads first; a wave's
// accesses are whole rows. Bound: memory (32.7 thousand positions of 4 heads
// from 8 bits: 169 MB in 25.5 us, 6.6 TB/s, four fifths of it stores).
constexpr int kReadRows = 2;
template <int HD, bool Q8>
__global__ __launch_bounds__(256) void read_kernel(KvDev kv, const int *__restrict__ slot, const int *__restrict__ posv,
                                                   int n_tok, float *__restrict__ k, float *__restrict__ v,
                                                   int64_t kv_stride) {
	constexpr int L = HD / 4, R = 256 / L;   // lanes of a row, rows of a workgroup at a time
	const uint32_t per = 2 * kv.kvh, t = threadIdx.x % L, row0 = blockIdx.x * (R * kReadRows) + threadIdx.x / L;
	float *dst[kReadRows];
	uint2 w[kReadRows];
	float sc[kReadRows];
#pragma unroll
	for (int i = 0; i < kReadRows; i++) {
		const uint32_t row = row0 + i * R;
		const int tok = (int)(row / per), h = (int)(row - tok * per), at = min(tok, n_tok - 1);
		const int sl = slot ? slot[at] : at, pos = posv[at];
		const bool is_v = h >= kv.kvh;
		float *to = is_v ? v : k;
		const bool on = tok < n_tok && to && sl >= 0 && sl < kv.n_slots && pos >= 0 && pos < kv.max_seq;
		const int hh = is_v ? h - kv.kvh : h;
		// (a row that is left out reads the cache's first)
		const size_t r = on ? ((size_t)sl * kv.kvh + hh) * kv.max_seq + pos : 0;
		dst[i] = on ? to + tok * kv_stride + (int64_t)hh * HD + 4 * t : nullptr;
		const uint8_t *src = (is_v ? kv.v : kv.k) + (r * HD + 4 * t) * (Q8 ? 1 : 2);
		if (Q8) w[i] = make_uint2(*(const uint32_t *)src, 0);
		else w[i] = *(const uint2 *)src;
		sc[i] = (is_v ? kv.vs : kv.ks)[r];
	}
#pragma unroll
	for (int i = 0; i < kReadRows; i++) {
		float x[4];
		if (Q8) {
#pragma unroll
			for (int j = 0; j < 4; j++) x[j] = (float)(int8_t)(w[i].x >> (8 * j)) * sc[i];
		} else {
			x[0] = f16_to_f32(w[i].x & 0xFFFFu) * sc[i];
			x[1] = f16_to_f32(w[i].x >> 16) * sc[i];
			x[2] = f16_to_f32(w[i].y & 0xFFFFu) * sc[i];
			x[3] = f16_to_f32(w[i].y >> 16) * sc[i];
		}
		if (dst[i]) put4_past(dst[i], x);
	}
}

int tokens_check(const hako_gpu_kv *kv, const int *slot, const int *pos, int n_tok) {
	if (n_tok < 0) return set_error(HAKO_GPU_EINVAL, "%d tokens", n_tok);
	if (!pos && n_tok) return set_error(HAKO_GPU_EINVAL, "null positions");
	if (!slot && n_tok > kv->n_slots)
		return set_error(HAKO_GPU_EINVAL, "%d tokens without slots in a cache of %d", n_tok, kv->n_slots);
	return HAKO_GPU_OK;
}

// workgroups for `rows` head rows, `each` of them to one
int row_blocks(int64_t rows, int each, dim3 *grid) {
	const int64_t n = (rows + each - 1) / each;
	if (n > kMaxThreads / 256) return set_error(HAKO_GPU_EINVAL, "%lld head rows in one call", (long long)rows);
	*grid = dim3((unsigned)n);
	return HAKO_GPU_OK;
}

}  // namespace
}  // namespace hako

using namespace hako;

extern "C" {

int hako_gpu_kv_bytes(const hako_gpu_kv *kv, size_t *codes, size_t *scales) {
	if (!codes || !scales) return set_error(HAKO_GPU_EINVAL, "null argument");
	if (int rc = kv_shape_check(kv)) return rc;
	const size_t rows = (size_t)kv->n_slots * kv->n_kv_heads * kv->max_seq;
	*codes = rows * kv->head_dim * kv_elt(kv->type);
	*scales = rows * sizeof(float);
	return ok();
}

int hako_gpu_kv_append(const hako_gpu_kv *kv, const int *slot, const int *pos, int n_tok, const float *k,
                       const float *v, int64_t kv_stride, const hako_gpu_rope *rope, const float *q, float *q_out,
                       int n_heads, int64_t q_stride, int64_t q_out_stride) {
	if (int rc = kv_check(kv)) return rc;
	if (int rc = tokens_check(kv, slot, pos, n_tok)) return rc;
	const int64_t kvw = (int64_t)kv->n_kv_heads * kv->head_dim;
	if (int rc = rows_check("k", k, kv_stride, kvw)) return rc;
	if (int rc = rows_check("v", v, kv_stride, kvw)) return rc;
	RopeDev r{nullptr, 0, 0, 0};
	if (rope) {
		if (!rope->table || ((uintptr_t)rope->table & 15) || rope->n_pos < 1 || rope->rot_dim < 8 ||
		    rope->rot_dim % 8 || rope->rot_dim > kv->head_dim || (rope->interleaved != 0 && rope->interleaved != 1))
			return set_error(HAKO_GPU_EINVAL,
			                 "rope: table %p (16-byte aligned), %d positions, rot_dim %d (a multiple of 8 up to %d), "
			                 "interleaved %d",
			                 (const void *)rope->table, rope->n_pos, rope->rot_dim, kv->head_dim, rope->interleaved);
		r = {rope->table, rope->n_pos, rope->rot_dim, rope->interleaved};
	}
	int H = 0;
	if (q || q_out) {
		if (!rope) return set_error(HAKO_GPU_EINVAL, "queries without a rotation");
		if (n_heads < 1 || n_heads > 65535) return set_error(HAKO_GPU_EINVAL, "%d query heads", n_heads);
		if (int rc = rows_check("q", q, q_stride, (int64_t)n_heads * kv->head_dim)) return rc;
		if (int rc = rows_check("q_out", q_out, q_out_stride, (int64_t)n_heads * kv->head_dim)) return rc;
		if (q == q_out && q_stride != q_out_stride)
			return set_error(HAKO_GPU_EINVAL, "queries rotated in place with two strides");
		H = n_heads;
	}
	if (int rc = require_device()) return rc;
	if (n_tok == 0) return ok();
	dim3 grid;
	if (int rc = row_blocks((int64_t)n_tok * (H + 2 * kv->n_kv_heads), 256 / (kv->head_dim / 8), &grid)) return rc;
#define HK_APPEND(HD, Q8)                                                                                          \
	hipLaunchKernelGGL((append_kernel<HD, Q8>), grid, dim3(256), 0, stream(), kv_dev(kv), slot, pos, n_tok, k, v,    \
	                   kv_stride, r, q, q_out, H, q_stride, q_out_stride)
	if (kv->head_dim == 128) {
		if (kv->type == HAKO_KV_Q8) HK_APPEND(128, true);
		else HK_APPEND(128, false);
	} else {
		if (kv->type == HAKO_KV_Q8) HK_APPEND(64, true);
		else HK_APPEND(64, false);
	}
#undef HK_APPEND
	HK_LAUNCHED("kv append");
	return ok();
}

int hako_gpu_kv_read(const hako_gpu_kv *kv, const int *slot, const int *pos, int n_tok, float *k, float *v,
                     int64_t kv_stride) {
	if (int rc = kv_check(kv)) return rc;
	if (int rc = tokens_check(kv, slot, pos, n_tok)) return rc;
	if (!k && !v) return set_error(HAKO_GPU_EINVAL, "neither keys nor values wanted");
	const int64_t kvw = (int64_t)kv->n_kv_heads * kv->head_dim;
	if (k)
		if (int rc = rows_check("k", k, kv_stride, kvw)) return rc;
	if (v)
		if (int rc = rows_check("v", v, kv_stride, kvw)) return rc;
	if (int rc = require_device()) return rc;
	if (n_tok == 0) return ok();
	dim3 grid;
	if (int rc = row_blocks((int64_t)n_tok * 2 * kv->n_kv_heads, 256 / (kv->head_dim / 4) * kReadRows, &grid)) return rc;
#define HK_READ(HD, Q8) \
	hipLaunchKernelGGL((read_kernel<HD, Q8>), grid, dim3(256), 0, stream(), kv_dev(kv), slot, pos, n_tok, k, v, kv_stride)
	if (kv->head_dim == 128) {
		if (kv->type == HAKO_KV_Q8) HK_READ(128, true);
		else HK_READ(128, false);
	} else {
		if (kv->type == HAKO_KV_Q8) HK_READ(64, true);
		else HK_READ(64, false);
	}
#undef HK_READ
	HK_LAUNCHED("kv read");
	return ok();
}

}  // extern "C"
