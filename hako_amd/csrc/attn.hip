// attn.hip — attention over the quantised cache (include/hako_attn.h): single
// tokens of many sequences, whole packed prompts, both also under a window with
// sinks, and trees of drafted tokens.
//
// One pass over the keys with a running maximum and sum (log2 units):
//   u_p = scale log2(e) q.k_p,  M = max u_p,  l = sum 2^(u_p - M),
//   o = sum 2^(u_p - M) v_p / l.
// Both products run on the fp16 matrix cores with fp32 sums and keep fp32
// accuracy: cache codes (int8 or half) are exact in fp16, and the fp32 factor
// (the query; the weight times the value row's scale) goes in as two halves,
// hi = its fp16 and lo = fp16 of the rest, 22 bits together. A query row is
// first scaled by a power of two that puts its maximum into [2^14, 2^15), the
// weights by one that puts them below 2^14, so that lo stays clear of the
// half's subnormals over 2^-14 of the maximum.
//
// Scores are formed transposed (S^T = K Q^T: lanes hold queries, registers
// keys), because then a lane's scores are, in its own registers, the operand
// of the second product (O^T = V^T P^T) and the running maximum, sum and
// rescaling belong to the lane; keys are dealt to the tile's rows so that a
// lane's registers are consecutive keys.
#include "kv.h"

#include <algorithm>
#include <float.h>
#include <math.h>
#include <new>
#include <stddef.h>
#include <vector>

// CALL(HD, Q8) for a cache's head size and type.
#define HK_KV_SWITCH(kv, CALL)                                     \
	((kv)->head_dim == 128 ? ((kv)->type == HAKO_KV_Q8 ? CALL(128, true) : CALL(128, false)) \
	                       : ((kv)->type == HAKO_KV_Q8 ? CALL(64, true) : CALL(64, false)))

namespace hako {
namespace {

constexpr int kMaxGroup = 16;    // query heads per key/value head
constexpr int kSeqs = 48;        // sequences of one prompt launch (by value in the kernel arguments)
constexpr int kItems = 480;      // items of a launch whose order the host sets (likewise)
constexpr int kWsAttn = 7;       // library workspace slot of the records
constexpr int kKeys = 64;        // keys per chunk of the tiled kernel
constexpr int kLongPart = 2048;  // keys of a part where sequences alone fill the chip
constexpr int kLongWindow = 8192; // the same under a window
constexpr int kWaves = 4;        // waves per workgroup of the direct and the single-token kernel
// M is a whole number not below what it was taken from (the maximum of the
// scores, in log2, plus the exponent of the value scales), so that what is
// rescaled when it moves, and where sums meet, is so by exact powers of two;
// it moves only when that passes it by kSlack, which is rare. From kBig on a
// float has no room for the exponent beside the score (see Base).
constexpr float kNone = -FLT_MAX;   // M of a row that has seen no key
constexpr float kBig = 4194304.0f;
constexpr float kUp = 6.0f;         // weights are 2^(u - M + 6): at most 2^14 while u <= M + kSlack
constexpr float kSlack = 8.0f;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

// prompts and trees: 1 = direct kernel, 2 and 3 = tiled kernel of 256 and 128 rows, 0 = by shape (tuning knob)
int g_attn_prompt = 0;

struct AttnKv {
	const uint8_t *k, *v;
	const float *ks, *vs;
	int n_slots, max_seq, kvh;
	int prefix_slot, prefix_len;
	int len_add;   // added to every length (single tokens)
	int window, sinks;   // a token's last positions and the first ones that stay (window 0: it sees every one before it)
};

// A prompt launch: sequence s has len[s] tokens from row row[s] of q and
// out, at positions start[s].. of slot[s]; items item[s].. of the grid are
// its tiles, the last tile first, each in nsplit[s] parts of its keys. The
// tiles of more than `unit` steps, whose parts are joined, hold the last
// join[s + 1] - join[s] tokens.
struct SeqTab {
	int n, tile_tokens, unit;   // tokens per tile, steps per part
	int row[kSeqs], len[kSeqs], slot[kSeqs], start[kSeqs], item[kSeqs + 1], nsplit[kSeqs];
	int join[kSeqs + 1];
	uint32_t rec[kSeqs];        // first record of a sequence's split tokens
};

// Positions that a tile of tokens looks at, in steps of K: those of [0, pend)
// of row r0's slot and head, n0 steps, then those of [b0, end) of r1's.
struct Span {
	size_t r0, r1;
	int pend, n0, b0, end;
	__device__ __forceinline__ bool first(int step) const { return step < n0; }
	template <int K>
	__device__ __forceinline__ int key(int step) const { return step < n0 ? K * step : b0 + K * (step - n0); }
	// positions from here on are not the step's
	__device__ __forceinline__ int top(int step) const { return step < n0 ? pend : end; }
};

// Which keys of a step a row sees: at(k, ..) turns to those from key k on,
// sees(i) tells of the i-th of them. lim: the row sees keys below it.
// Every one:
struct Below {
	static constexpr bool kHi = false, kBlanks = false;
	int lim;
	__device__ __forceinline__ void at(int k, int top, bool) { lim = min(lim, top) - k; }
	__device__ __forceinline__ bool sees(int i) const { return i < lim; }
	// whether keys before k are of use to rows of the least lim lo (those from k on may be)
	__device__ __forceinline__ bool reaches(int, bool, int) const { return true; }
	// whether a step of K keys at k needs the mask; lo, hi: the least and greatest lim of the rows
	template <int K>
	__device__ __forceinline__ bool masks(int k, int top, bool, int lo, int) const { return k + K > min(lo, top); }
};
// The last `window`, and in a span's first steps every one:
struct Within {
	static constexpr bool kHi = true, kBlanks = false;
	int lim, window, from;
	__device__ __forceinline__ void at(int k, int top, bool first) {
		from = first ? 0 : lim - window - k;
		lim = min(lim, top) - k;
	}
	__device__ __forceinline__ bool sees(int i) const { return i < lim && i >= from; }
	__device__ __forceinline__ bool reaches(int k, bool first, int lo) const { return first || k > lo - window; }
	template <int K>
	__device__ __forceinline__ bool masks(int k, int top, bool first, int lo, int hi) const {
		return k + K > min(lo, top) || (!first && k < hi - window);
	}
};
// Those below lim, and of the 64 from there on those of its bits (any: all rows' bits, the same in every lane):
struct Nodes {
	static constexpr bool kHi = false, kBlanks = true;
	int lim;
	uint64_t bits, any, w;
	// the 64 keys from k on as bits: those below lim, then those of m
	__device__ __forceinline__ uint64_t from(int k, uint64_t m) const {
		const int s = k - lim;
		if (s >= 0) return s < 64 ? m >> s : 0;
		return s > -64 ? m << -s | ((1ull << -s) - 1) : ~0ull;
	}
	__device__ __forceinline__ void at(int k, int top, bool) {
		const int n = top - k;
		w = from(k, bits);
		w = n >= 64 ? w : n > 0 ? w & ((1ull << n) - 1) : 0;
	}
	__device__ __forceinline__ bool sees(int i) const { return w >> i & 1; }
	__device__ __forceinline__ bool reaches(int, bool, int) const { return true; }
	template <int K>
	__device__ __forceinline__ bool masks(int k, int top, bool, int lo, int) const { return k + K > min(lo, top); }
	// whether a step of K keys at k may hold rows that nobody sees, which may never have been written; those that are not
	template <int K>
	__device__ __forceinline__ bool gaps(int k) const { return k + K > lim; }
	__device__ __forceinline__ uint64_t written(int k) const { return from(k, any); }
};

// The same value, made anew where this stands: addresses and masks that
// follow from it are computed there rather than held in registers across a
// loop.
__device__ __forceinline__ int fresh(int v) {
	asm volatile("" : "+v"(v));
	return v;
}

// What a wave wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync() {
	__builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
	__builtin_amdgcn_wave_barrier();
	__builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// What a row's sums are taken against, M in two parts: weights are
// 2^(u - m - e + kUp). A small base, |m| < kBig, has e = 0 and the exponent of
// the value scales in m. A big one has the score's whole number in m and that
// exponent in e: past 2^24 m + e would round to m (as would kUp), and weights
// times value scales leave a half's range (before this was so, keys of 2^30
// and values of 2^17 gave infinities). Steps with a big base go through a
// block of their own, out of the way of the others, whose times stayed the same.
struct Base {
	float m, e;
	__device__ __forceinline__ bool big() const { return (e != 0.0f || __builtin_fabsf(m) >= kBig) && m != kNone; }
};
// How far a lies above b, in powers of two: exact where they are near.
__device__ __forceinline__ float above(Base a, Base b) { return (a.m - b.m) + (a.e - b.e); }
// The same for ldexp, of sums that move from a to b >= a: any power of two, and to 0 from kNone.
__device__ __forceinline__ int steps_down(Base a, Base b) { return (int)__builtin_fmaxf(above(a, b), -1000.0f); }

// The sums of part of a row's keys: value sums o [record][HD], (M, l) in ml, and where e is not 0, which l's sign tells,
// e (so that nobody reads it who need not).
struct Records {
	float *o;
	float2 *ml;
	float *e;
	__device__ __forceinline__ void put(size_t r, Base b, float l) const {
		ml[r] = make_float2(b.m, b.e != 0.0f ? -__builtin_fabsf(l) : __builtin_fabsf(l));
		if (b.e != 0.0f) e[r] = b.e;
	}
};
__device__ __forceinline__ bool has_e(float2 ml) { return __builtin_bit_cast(int, ml.y) < 0; }
__device__ __forceinline__ Base base_of(float2 ml, const float *e) { return {ml.x, has_e(ml) ? *e : 0.0f}; }

// Whether a step moves a small base M up, ue being the row's largest score there plus the exponent of the value scales.
__device__ __forceinline__ bool passes(float ue, float M) { return ue > M + kSlack; }
// ... and to a big one.
__device__ __forceinline__ bool passes_big(float ue, float M) { return passes(ue, M) && !(__builtin_fabsf(__builtin_ceilf(ue)) < kBig); }
// Moves a small base that stays small: the shift of the row's sums.
__device__ __forceinline__ int move_up(float &M, float ue) {
	const float n = passes(ue, M) ? __builtin_ceilf(ue) : M;
	const int f = steps_down({M, 0.0f}, {n, 0.0f});
	M = n;
	return f;
}
// Moves any base: u is the largest score, e the exponent of the value scales, ue their sum. Small bases go as in
// move_up, so that a row's answer is its own whatever the others of its wave do.
__device__ __forceinline__ int move_up_any(Base &b, float u, float e, float ue) {
	Base n = b;
	if (b.big() ? (u - b.m) + (e - b.e) > kSlack : passes(ue, b.m)) {
		const float c = __builtin_ceilf(ue);
		n = __builtin_fabsf(c) < kBig ? Base{c, 0.0f} : Base{__builtin_ceilf(u), e};
	}
	const int f = steps_down(b, n);
	b = n;
	return f;
}
// N scores (in units of esc) against a big base: those whose weights are exp2(score esc). (esc is a power of two, and a
// score that overflows here lies far below the base.)
template <int N, class V>
__device__ __forceinline__ void big_scores(V &sc, Base b, float esc) {
	const float inv = __builtin_bit_cast(float, 0x7F000000u - __builtin_bit_cast(uint32_t, esc));   // 1 / esc
#pragma unroll
	for (int i = 0; i < N; i++) {
		const float w = (__builtin_fmaf(sc[i], esc, -b.m) + (kUp - b.e)) * inv;
		sc[i] = b.big() ? w : sc[i];
	}
}

// Four int8 codes as halves: byte + 128 under the exponent byte 0x64 is the
// half 1024 + (code + 128).
__device__ __forceinline__ h2 bytes_h2(uint32_t biased, uint32_t sel) {
	const h2 t = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, biased, sel));
	return t - (h2){(_Float16)1152.0f, (_Float16)1152.0f};
}
constexpr uint32_t kLo2 = 0x04010400u, kHi2 = 0x04030402u;
constexpr uint32_t kFlip = 0x80808080u;

// fp32 pair -> hi halves (toward zero; the rest is exact) and lo halves.
__device__ __forceinline__ void split2(float a, float b, h2 &hi, h2 &lo) {
	hi = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
	lo = (h2){(_Float16)(a - (float)hi.x), (_Float16)(b - (float)hi.y)};
}

// A power of two that brings a row of queries with maximum a to [2^14, 2^15).
__device__ __forceinline__ int row_exp(float a) { return f16_split_exp(a) - 14; }

// Eight queries scaled by 2^-e as hi and lo halves (each rounded to nearest).
__device__ __forceinline__ void split_q(const float *x, int e, h8 &hi, h8 &lo) {
#pragma unroll
	for (int j = 0; j < 8; j++) {
		const float f = __builtin_ldexpf(x[j], -e);
		hi[j] = (_Float16)f;
		lo[j] = (_Float16)(f - (float)hi[j]);
	}
}

// The exponent of the largest value scale of some keys. It goes into M, which
// is not below any u_p + exponent of key p's step: weights times value scales
// then fit a half whatever the scales are. Only scales that a row sees count
// for it (those of a later token may be larger by any factor). Not below -88:
// l, up to 2^(14 + 88) a key, stays finite.
__device__ __forceinline__ float scale_exp(float vmax) {
	return (float)max((int)(__builtin_bit_cast(uint32_t, vmax) >> 23) - 127, -88);
}

// ── tiled kernel: 256 query rows against chunks of 64 keys ──
//
// Rows are (token, head of the group) pairs, token-major, so that one staged
// chunk serves every query head of a key/value head. Eight waves of 32 rows
// (v_mfma_f32_32x32x16_f16); per chunk the workgroup converts the codes to
// halves in LDS, keys as [key][dim] and values transposed as [dim][key], so
// that every operand is one 16-byte LDS read. Two LDS buffers, one barrier per
// chunk.
//
// Bound: matrix work at the chip's power. 8192 tokens of 7B heads (28 / 4 of
// 128, 481 GFLOP, each product twice: 962) take 0.84-0.86 ms, 1.1 PFLOP/s of
// matrix operations; an 8192^3 fp16 product of the library runs at 1.09 here.
// The matrix pipes are then busy 64% of the cycles, the vector pipes 59%, at
// 1.8 GHz. On the way (the same call): 128-row tiles and one accumulator set
// per masked and unmasked instance 1.51 ms; one instance, 16-byte LDS reads
// 1.00; the weights of the second 32 keys formed under the values' products of
// the first 0.95; 256 rows to a chunk 0.94; padded rows, no address arithmetic
// in the loop 0.90 (868 against 907 us on one box); staging at opposite ends
// of a chunk by a SIMD's two waves 0.84. No difference: wave priorities around
// either product, reads left to the compiler's own order (871 against 869).
// Queries and outputs pass through LDS in whole lines, the first chunk's codes
// on their way meanwhile: an item's start and end 13 us, 16 before (packed
// prompts of 4097 tokens 92 us, 97; 8192 tokens under a window of 128 107, 123).
//
// Tiles of 128 rows and four waves, two workgroups a CU, stage each chunk for
// half as many rows: for windows, whose tiles are short and much alike, where
// half a round of items saves more (see window_kernel), and for small drafted
// trees. Under a window a tile
// passes the chunks of the sinks and those from its first token's window on,
// and masks the chunks at either border alone: 16384 tokens under 4096 take
// 1.45 ms on the fastest box seen, 1.16 PFLOP/s of matrix operations, matrix
// pipes busy 63% of the cycles.

// Rows in LDS are padded by 16 bytes, so that lanes on consecutive rows meet
// different banks. A chunk's keys lie in the order of the score tiles' rows
// (key_row), its value dims with equal dim % 4 together (dim_row): both let
// the lanes that write a chunk, and those that read it, go row by row.
template <int HD>
constexpr int kKeyRow = 2 * HD + 16;
constexpr int kDimRow = 2 * kKeys + 16;
// Row of a key: tile row 8 a + 4 h + b holds key 16 (a>>1) + 8 h + 4 (a&1) + b
// (of its 32), so that register v of lane half h is key 16 (v>>3) + 8 h + (v&7).
__device__ __forceinline__ int key_row(int key) { return (key & ~12) | ((key >> 1) & 4) | ((key << 1) & 8); }
template <int HD>
__device__ __forceinline__ int dim_row(int dim) { return (dim & 3) * (HD / 4) + (dim >> 2); }

template <int HD, bool Q8, int W>
struct Stage {
	static constexpr int EB = Q8 ? 1 : 2, NT = 64 * W;
	static constexpr int KU = kKeys * HD * EB / 16, KL = (KU + NT - 1) / NT;   // 16-byte key loads of a chunk, per thread
	static constexpr int VQ = HD / 4, VK = 4;                                  // dim quads; a thread takes 4 keys x 4 dims
	static constexpr int VT = kKeys / VK * VQ, VL = (VT + NT - 1) / NT;        // such pieces of the values (512 or 256), per thread
	uint4 k[KL];
	uint32_t v[VL][VK][EB];
	float ks, vs;

	__device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t vr, __amdgpu_buffer_rsrc_t ksr,
	                                     __amdgpu_buffer_rsrc_t vsr, int key0, int tid) {
#pragma unroll
		for (int i = 0; i < KL; i++) {
			const int u = tid + NT * i;   // 16-byte unit of the chunk
			k[i] = ld_b128(kr, KU % NT && u >= KU ? kBufNone : (uint32_t)key0 * (HD * EB) + 16u * u);
		}
#pragma unroll
		for (int i = 0; i < VL; i++)
			if (VT % NT == 0 || tid < VT) {
				const int d = (tid + NT * i) % VQ, kg = (tid + NT * i) / VQ;
				const uint32_t off = ((uint32_t)(key0 + VK * kg) * HD + 4 * d) * EB;
#pragma unroll
				for (int j = 0; j < VK; j++) {
					if (Q8) v[i][j][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, (int)(off + j * HD), 0, 0);
					else {
						const uint2 t = ld_b64(vr, off + j * HD * 2);
						v[i][j][0] = t.x;
						v[i][j][EB - 1] = t.y;
					}
				}
			}
		if (tid < kKeys) {
			ks = ld_f32(ksr, 4u * (uint32_t)(key0 + tid));
			vs = ld_f32(vsr, 4u * (uint32_t)(key0 + tid));
		}
	}

	// Values of rows that nobody sees become zeros: halves there may be infinite or NaN, which a weight of 0 does not take
	// away. (Their scores are masked. Codes of 8 bits are finite whatever they are.)
	__device__ __forceinline__ void keep(uint64_t written, int tid) {
#pragma unroll
		for (int i = 0; i < VL; i++) {
			const uint32_t m = (uint32_t)(written >> (VK * ((tid + NT * i) / VQ) & 63));
#pragma unroll
			for (int j = 0; j < VK; j++)
#pragma unroll
				for (int w = 0; w < EB; w++) v[i][j][w] &= (uint32_t)__builtin_amdgcn_sbfe((int)m, j, 1);
		}
	}

	// Converted into LDS: keys k_s [64][HD], values v_s [HD][64] halves, the
	// scales and the exponent of the largest value scale.
	__device__ __forceinline__ void store(uint8_t *k_s, uint8_t *v_s, float *ks_s, float *vs_s, float *e_s, int tid) {
#pragma unroll
		for (int i = 0; i < KL; i++) {
			const int u = tid + NT * i;
			if (KU % NT && u >= KU) break;
			if (Q8) {
				const int key = u / (HD / 16), c = u % (HD / 16);
				const uint32_t w[4] = {k[i].x ^ kFlip, k[i].y ^ kFlip, k[i].z ^ kFlip, k[i].w ^ kFlip};
#pragma unroll
				for (int h = 0; h < 2; h++) {
					const h2 a = bytes_h2(w[2 * h], kLo2), b = bytes_h2(w[2 * h], kHi2);
					const h2 c2 = bytes_h2(w[2 * h + 1], kLo2), d = bytes_h2(w[2 * h + 1], kHi2);
					*(h8 *)(k_s + key_row(key) * kKeyRow<HD> + 32 * c + 16 * h) =
					    (h8){a.x, a.y, b.x, b.y, c2.x, c2.y, d.x, d.y};
				}
			} else {
				const int key = u / (HD / 8), c = u % (HD / 8);
				*(uint4 *)(k_s + key_row(key) * kKeyRow<HD> + 16 * c) = k[i];
			}
		}
#pragma unroll
		for (int n = 0; n < VL; n++) {
			if (VT % NT && tid >= VT) break;
			const int d = (tid + NT * n) % VQ, kg = (tid + NT * n) / VQ;
			h2 t[4][VK / 2];   // [dim][key pair]
#pragma unroll
			for (int p = 0; p < VK / 2; p++) {
				if (Q8) {
					const uint32_t a = v[n][2 * p][0] ^ kFlip, b = v[n][2 * p + 1][0] ^ kFlip;
					const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u), hi = __builtin_amdgcn_perm(b, a, 0x07030602u);
					t[0][p] = bytes_h2(lo, kLo2);
					t[1][p] = bytes_h2(lo, kHi2);
					t[2][p] = bytes_h2(hi, kLo2);
					t[3][p] = bytes_h2(hi, kHi2);
				} else {
#pragma unroll
					for (int w = 0; w < 2; w++) {
						const uint32_t a = v[n][2 * p][w * (EB - 1)], b = v[n][2 * p + 1][w * (EB - 1)];
						t[2 * w][p] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x05040100u));
						t[2 * w + 1][p] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x07060302u));
					}
				}
			}
#pragma unroll
			for (int i = 0; i < 4; i++) {
				const int dim = 4 * d + i;
				*(uint2 *)(v_s + dim_row<HD>(dim) * kDimRow + 2 * VK * kg) =
				    make_uint2(__builtin_bit_cast(uint32_t, t[i][0]), __builtin_bit_cast(uint32_t, t[i][1]));
			}
		}
		if (tid < kKeys) {
			// a value row that is not finite makes its scores NaN, which a row that may not see it masks
			const bool fin = __builtin_isfinite(vs);
			vs = fin ? vs : 0.0f;
			const float e = scale_exp(wave_max(__builtin_fabsf(vs)));
			ks_s[tid] = fin ? ks : __builtin_nanf("");
			vs_s[tid] = vs;
			if (tid == 0) *e_s = e;
		}
	}
};

// One wave's 32 rows over the chunks of a part. lim: the lane's row sees keys
// (positions) below it; out: O^T (value sums), M and l.
template <int HD, bool Q8, int W>
struct Tile {
	static constexpr int KS = HD / 16, DT = HD / 32;
	static constexpr int kKB = kKeys * kKeyRow<HD>, kVB = HD * kDimRow;
	struct Lds {
		alignas(16) uint8_t k[2][kKB];
		alignas(16) uint8_t v[2][kVB];
		alignas(16) float ks[2][kKeys];
		alignas(16) float vs[2][kKeys];
		float e[2];
		float be[64 * W];   // e of the rows' bases
	};
	h8 qh[KS], ql[KS];
	float esc;      // 2^e of the row
	f16v o[DT];
	float M, l;
	uint64_t big;   // lanes whose base is big; while there are any, every lane's e is in LDS, else it is 0

	// The lane's row q (null: an idle row), times scale log2(e). Rows come as whole lines, half of the dims at a time
	// through LDS, the chunks' place.
	__device__ __forceinline__ void query(const float *q, float scale, Lds &lds, int tid) {
		constexpr int L = HD / 8, R = 2 * HD + 16;
		const int lane = tid & 63, h = lane >> 5;
		uint8_t *buf = lds.k[0] + (tid >> 6) * (32 * R);
		const uint64_t at = (uint64_t)(uintptr_t)q;
		float x[KS * 8], a = 0.0f;
		float4 y[L];
#pragma unroll
		for (int j = 0; j < L; j++) {
			const int row = j % (L / 2) * (64 / L) + lane / L;
			const uint64_t from = (uint64_t)(uint32_t)__shfl((int)(uint32_t)at, row) | ((uint64_t)(uint32_t)__shfl((int)(at >> 32), row) << 32);
			y[j] = make_float4(0, 0, 0, 0);
			if (from) y[j] = *(const float4 *)((const float *)(uintptr_t)from + HD / 2 * (j / (L / 2)) + 4 * (lane % L));
		}
#pragma unroll
		for (int p = 0; p < 2; p++) {
#pragma unroll
			for (int j = 0; j < L / 2; j++) *(float4 *)(buf + (j * (64 / L) + lane / L) * R + 16 * (lane % L)) = y[p * (L / 2) + j];
			wave_sync();
#pragma unroll
			for (int s = 0; s < KS / 2; s++) {
				const float4 u = *(const float4 *)(buf + (lane & 31) * R + 64 * s + 32 * h), w = *(const float4 *)(buf + (lane & 31) * R + 64 * s + 32 * h + 16);
				const float z[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
				for (int j = 0; j < 8; j++) {
					x[8 * (p * (KS / 2) + s) + j] = z[j] * scale;
					a = __builtin_fmaxf(a, __builtin_fabsf(z[j] * scale));
				}
			}
			wave_sync();
		}
		a = __builtin_fmaxf(a, __shfl_xor(a, 32));
		const int e = row_exp(a);
		esc = __builtin_ldexpf(1.0f, e);
#pragma unroll
		for (int s = 0; s < KS; s++) split_q(x + 8 * s, e, qh[s], ql[s]);
		clear();
		big = 0;
	}

	// The 64 keys of the chunk in LDS buffer `b`; mask: some row of the wave does not see all of them, see (at the lane
	// half's first key) tells which. (Two instances of this, with and without the mask, cost a second set of the value sums' registers.)
	// The weights of the second 32 keys form while the matrix cores add up the values of the first.
	template <class See>
	__device__ __forceinline__ void chunk(Lds &s, int b, bool mask, const See &see, int lane) {
		lane = fresh(lane);
		const int h = lane >> 5, i = lane & 31;
		const uint8_t *kr = s.k[b] + i * kKeyRow<HD> + 16 * h;
		f16v sc[2];
#pragma unroll
		for (int v = 0; v < 16; v++) sc[0][v] = sc[1][v] = 0.0f;
#pragma unroll
		for (int k = 0; k < KS; k++)
#pragma unroll
			for (int t = 0; t < 2; t++) {
				const h8 a = *(const h8 *)(kr + 32 * t * kKeyRow<HD> + 32 * k);
				sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[k], sc[t], 0, 0, 0);
				sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[k], sc[t], 0, 0, 0);
			}
		feed<2 * KS>();
		__builtin_amdgcn_sched_barrier(0);
		float mx = -INFINITY;
#pragma unroll
		for (int t = 0; t < 2; t++)
#pragma unroll
			for (int g = 0; g < 4; g++) {
				const float4 ks = *(const float4 *)(s.ks[b] + 32 * t + 16 * (g >> 1) + 8 * h + 4 * (g & 1));
				const float kv[4] = {ks.x, ks.y, ks.z, ks.w};
#pragma unroll
				for (int j = 0; j < 4; j++) sc[t][4 * g + j] *= kv[j];
			}
		float e = s.e[b];
		if (mask) {
			float vm = 0.0f;
#pragma unroll
			for (int t = 0; t < 2; t++)
#pragma unroll
				for (int g = 0; g < 4; g++) {
					const float4 vs = *(const float4 *)(s.vs[b] + 32 * t + 16 * (g >> 1) + 8 * h + 4 * (g & 1));
					const float vv[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
					for (int j = 0; j < 4; j++) {
						const bool sees = see.sees(32 * t + 16 * (g >> 1) + 4 * (g & 1) + j);
						sc[t][4 * g + j] = sees ? sc[t][4 * g + j] : -INFINITY;
						vm = __builtin_fmaxf(vm, sees ? __builtin_fabsf(vv[j]) : 0.0f);
					}
				}
			e = scale_exp(__builtin_fmaxf(vm, __shfl_xor(vm, 32)));
		}
#pragma unroll
		for (int v = 0; v < 16; v++) mx = __builtin_fmaxf(__builtin_fmaxf(sc[0][v], sc[1][v]), mx);
		mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
		const float ue = __builtin_fmaf(mx, esc, e);
		float c = kUp - M;
		if (__ballot(passes(ue, M)) | big) {
			int f;
			if (__builtin_expect((__ballot(passes_big(ue, M)) | big) != 0, 0)) {
				Base at = {M, big ? s.be[threadIdx.x] : 0.0f};
				f = move_up_any(at, mx * esc, e, ue);
				M = at.m;
				s.be[threadIdx.x] = at.e;
				big = __ballot(at.big());
				big_scores<16>(sc[0], at, esc);
				big_scores<16>(sc[1], at, esc);
				c = at.big() ? 0.0f : kUp - M;
			} else {
				f = move_up(M, ue);
				c = kUp - M;
			}
			l = __builtin_ldexpf(l, f);
#pragma unroll
			for (int d = 0; d < DT; d++)
#pragma unroll
				for (int v = 0; v < 16; v++) o[d][v] = __builtin_ldexpf(o[d][v], f);
		}
		h8 ph[2][2], pl[2][2];
		weigh(s, b, 0, sc[0], c, h, ph[0], pl[0]);
		weigh(s, b, 1, sc[1], c, h, ph[1], pl[1]);
		add(s, b, 0, i, h, ph[0], pl[0]);
		add(s, b, 1, i, h, ph[1], pl[1]);
		__builtin_amdgcn_sched_barrier(0);
	}

	// Scores -> weights times the value scales, as halves, and their sum.
	__device__ __forceinline__ void weigh(const Lds &s, int b, int t, const f16v &sc, float c, int h, h8 ph[2], h8 pl[2]) {
#pragma unroll
		for (int g = 0; g < 4; g++) {
			const float4 vs = *(const float4 *)(s.vs[b] + 32 * t + 16 * (g >> 1) + 8 * h + 4 * (g & 1));
			const float vv[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
			for (int j = 0; j < 4; j += 2) {
				const float p0 = exp2_(__builtin_fmaf(sc[4 * g + j], esc, c)), p1 = exp2_(__builtin_fmaf(sc[4 * g + j + 1], esc, c));
				l += p0;
				l += p1;
				h2 a, d;
				split2(p0 * vv[j], p1 * vv[j + 1], a, d);
				ph[g >> 1][4 * (g & 1) + j] = a.x;
				ph[g >> 1][4 * (g & 1) + j + 1] = a.y;
				pl[g >> 1][4 * (g & 1) + j] = d.x;
				pl[g >> 1][4 * (g & 1) + j + 1] = d.y;
			}
		}
	}

	// o += the values of 32 keys times their weights.
	__device__ __forceinline__ void add(const Lds &s, int b, int t, int i, int h, const h8 ph[2], const h8 pl[2]) {
#pragma unroll
		for (int k = 0; k < 2; k++)
#pragma unroll
			for (int d = 0; d < DT; d++) {
				const h8 a = *(const h8 *)(s.v[b] + (32 * d + i) * kDimRow + 64 * t + 32 * k + 16 * h);
				o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[k], o[d], 0, 0, 0);
				o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[k], o[d], 0, 0, 0);
			}
	}

	// N operand reads from LDS, two products each: the reads three ahead of their products.
	template <int N>
	static __device__ __forceinline__ void feed() {
		__builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
		for (int i = 0; i < N; i++) {
			__builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
			if (i + 3 < N) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
		}
	}

	// Chunks [c0, c1) of a tile's span for the queries that ask() takes up while the first chunk's codes are on their
	// way. lo, hi: the least and greatest lim of the wave's rows.
	template <class See, class Ask>
	__device__ __forceinline__ void chunks(const AttnKv &c, const Span &sp, int c0, int c1, const See &row, int lo, int hi, Lds &s,
	                                       int tid, Ask ask) {
		constexpr int EB = Q8 ? 1 : 2;
		const int lane = tid & 63;
		Stage<HD, Q8, W> st;
		auto load = [&](int ch) {
			const size_t r = sp.first(ch) ? sp.r0 : sp.r1;
			const uint32_t n = (uint32_t)sp.top(ch);   // rows past it read as zeros
			st.load(stream_rsrc(uniform_ptr(c.k + r * HD * EB), n * HD * EB), stream_rsrc(uniform_ptr(c.v + r * HD * EB), n * HD * EB),
			        stream_rsrc(uniform_ptr(c.ks + r), n * 4), stream_rsrc(uniform_ptr(c.vs + r), n * 4), sp.key<kKeys>(ch), fresh(tid));
		};
		auto store = [&](int ch, int b) {
			if constexpr (See::kBlanks && !Q8)
				if (const int key0 = sp.key<kKeys>(ch); row.template gaps<kKeys>(key0)) st.keep(row.written(key0), fresh(tid));
			st.store(s.k[b], s.v[b], s.ks[b], s.vs[b], &s.e[b], fresh(tid));
		};
		// A wave's registers hold the codes two chunks on from the buffer that is read. The waves of a SIMD (w, w + 4)
		// put them into LDS at opposite ends of a chunk, so that one has vector work while the other has matrix work.
		if (c0 < c1) load(c0);
		__builtin_amdgcn_sched_barrier(0);
		ask();
		__syncthreads();
		if (c0 < c1) {
			store(c0, 0);
			if (c0 + 1 < c1) load(c0 + 1);
		}
		const bool early = __builtin_amdgcn_readfirstlane(tid >> 6) >= 4;
		__syncthreads();
		for (int ch = c0; ch < c1; ch++) {
			const int b = (ch - c0) & 1;
			auto stage = [&] {
				if (ch + 1 < c1) store(ch + 1, b ^ 1);
				if (ch + 2 < c1) load(ch + 2);
				__builtin_amdgcn_sched_barrier(0);
			};
			if (early) stage();
			const bool first = sp.first(ch);
			const int key0 = sp.key<kKeys>(ch), top = sp.top(ch);
			if (key0 < min(hi, top) && row.reaches(key0 + kKeys, first, lo)) {   // some row of the wave sees some of these keys
				See see = row;
				see.at(key0 + 8 * (fresh(lane) >> 5), top, first);
				chunk(s, b, row.template masks<kKeys>(key0, top, first, lo, hi), see, lane);
			}
			if (!early) stage();
			__syncthreads();
		}
		l += __shfl_xor(l, 32);
	}

	// A row that has seen nothing.
	__device__ __forceinline__ void clear() {
#pragma unroll
		for (int d = 0; d < DT; d++)
#pragma unroll
			for (int v = 0; v < 16; v++) o[d][v] = 0.0f;
		M = kNone;
		l = 0.0f;
	}

	// The rows' value sums times f to their places, dst for the lane's (null: nowhere): row 8 a + 4 h + b of tile d is
	// dim_row 32 d + .. Half of the dims at a time pass through LDS, the chunks' place, so that stores are of whole lines
	// (a lane's own stores, 16 bytes to each of 64 rows, took 5 us of an item of 148, these 1.5).
	__device__ __forceinline__ void put(float *dst, float f, Lds &s, int tid) const {
		constexpr int L = HD / 8, R = 2 * HD + 16, NV = 2 * DT;
		static_assert(W * 32 * R <= 2 * kKB + 2 * kVB && offsetof(Lds, v) == 2 * kKB, "rows in the place of the chunks");
		const int lane = tid & 63, i = lane & 31, h = lane >> 5;
		uint8_t *buf = s.k[0] + (tid >> 6) * (32 * R);
		const uint64_t at = (uint64_t)(uintptr_t)dst;
#pragma unroll
		for (int p = 0; p < 2; p++) {
#pragma unroll
			for (int v = NV * p; v < NV * p + NV; v++) {
				const int r = 8 * (v >> 2) + 4 * h + (v & 3) - HD / 8 * p;   // quad of dims
				*(float4 *)(buf + i * R + 16 * r) = DT == 4 ? make_float4(o[0][v] * f, o[1][v] * f, o[2 % DT][v] * f, o[3 % DT][v] * f)
				                                            : make_float4(o[0][v] * f, o[0][v + 8] * f, o[1][v] * f, o[1][v + 8] * f);
			}
			wave_sync();
#pragma unroll
			for (int j = 0; j < L / 2; j++) {
				const int row = j * (64 / L) + lane / L;
				const float4 x = *(const float4 *)(buf + row * R + 16 * (lane % L));
				const uint64_t to = (uint64_t)(uint32_t)__shfl((int)(uint32_t)at, row) | ((uint64_t)(uint32_t)__shfl((int)(at >> 32), row) << 32);
				if (to) *(float4 *)((float *)(uintptr_t)to + HD / 2 * p + 4 * (lane % L)) = x;
			}
			wave_sync();
		}
	}
};

__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
	for (int k = 1; k < 64; k <<= 1) v = min(v, __shfl_xor(v, k));
	return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
	for (int k = 1; k < 64; k <<= 1) v = max(v, __shfl_xor(v, k));
	return __builtin_amdgcn_readfirstlane(v);
}

// Steps of K keys of a tile that sees positions below `end`: the prefix's, then its own.
template <int K>
__host__ __device__ __forceinline__ int tile_steps(int end, int prefix) {
	const int p = prefix < end ? prefix : end;
	return (p + K - 1) / K + (end - p + K - 1) / K;
}

// What a launch's tokens see.
struct Reach {
	int prefix, window, sinks;
};
// Steps of a tile of `tokens` tokens from position `first` (as if it were full: the steps of a sequence's tiles then never
// fall), the last of them at end - 1. With a window whose last token leaves some positions past the sinks behind these are
// the sinks' and those from the first token's window on; else all before it.
__host__ __device__ __forceinline__ bool two_spans(const Reach &r, int first, int tokens) { return first + tokens - r.window > r.sinks; }
__host__ __device__ __forceinline__ int span_start(const Reach &r, int first) {
	return first - r.window + 1 > r.sinks ? first - r.window + 1 : r.sinks;
}
template <int K, bool WIN>
__host__ __device__ __forceinline__ int reach_steps(const Reach &r, int first, int tokens, int end) {
	if (!WIN) return tile_steps<K>(end, r.prefix);
	const int e = first + tokens;
	if (!two_spans(r, first, tokens)) return (e + K - 1) / K;
	return (r.sinks + K - 1) / K + (e - span_start(r, first) + K - 1) / K;
}
template <int K, bool WIN>
__device__ __forceinline__ Span span_of(const AttnKv &c, int kvh, int slot, int first, int tokens, int end) {
	auto base = [&](int sl) { return ((size_t)sl * c.kvh + kvh) * c.max_seq; };
	if (!WIN) {
		const int pend = min(c.prefix_len, end);
		return {base(c.prefix_len > 0 ? c.prefix_slot : slot), base(slot), pend, (pend + K - 1) / K, c.prefix_len, end};
	}
	const Reach r = {0, c.window, c.sinks};
	const bool two = two_spans(r, first, tokens);
	const int s = two ? c.sinks : first + tokens;   // what every token sees of what comes before it
	return {base(slot), base(slot), min(s, end), (s + K - 1) / K, two ? span_start(r, first) : end, end};
}

// The items of a launch, the longest first: sequence << 26 | tile << 8 | part.
// Without (n 0) they go by sequence, tile and part.
struct ItemTab {
	int n;
	uint32_t item[kItems];
};

// What a workgroup of a prompt launch works on. A tile of nc steps is
// ceil(nc / unit) parts of equal length.
struct Item {
	int sq, slot, tok0, ntok, end, part, parts, c0, c1;
};
template <int K, bool WIN>
__device__ __forceinline__ bool item_of(const SeqTab &t, const ItemTab *order, int item, const Reach &reach, Item &x) {
	int tile;
	if (order && order->n) {
		const uint32_t v = order->item[item];
		x.sq = (int)(v >> 26);
		tile = (int)((v >> 8) & 0x3FFFFu);
		x.part = (int)(v & 0xFFu);
	} else {
		x.sq = 0;
		while (item >= t.item[x.sq + 1]) x.sq++;
		const int ns = t.nsplit[x.sq], it = item - t.item[x.sq];
		tile = (t.len[x.sq] + t.tile_tokens - 1) / t.tile_tokens - 1 - it / ns;
		x.part = it % ns;
	}
	x.slot = t.slot[x.sq];
	x.tok0 = tile * t.tile_tokens;
	x.ntok = min(t.tile_tokens, t.len[x.sq] - x.tok0);
	x.end = t.start[x.sq] + x.tok0 + x.ntok;
	const int nc = reach_steps<K, WIN>(reach, t.start[x.sq] + x.tok0, t.tile_tokens, x.end);
	x.parts = (nc + t.unit - 1) / t.unit;
	const int per = (nc + x.parts - 1) / x.parts;
	x.c0 = x.part * per;
	x.c1 = min(nc, x.c0 + per);
	return x.part < x.parts;
}
// Record of a split token's query head and part.
__device__ __forceinline__ size_t record_of(const SeqTab &t, const Item &x, int tok, int H, int head) {
	const int first = t.len[x.sq] - (t.join[x.sq + 1] - t.join[x.sq]);   // the first split token
	return (size_t)t.rec[x.sq] + ((size_t)(x.tok0 + tok - first) * H + head) * t.nsplit[x.sq] + x.part;
}

// ── direct kernel: 32 query rows, the keys dealt to the waves ──
//
// The same products on 32 rows, but each wave takes its own steps of 32 keys
// with the codes straight from memory in the operands' registers (keys as they
// lie; values paired by byte permutes), and the waves meet once, in LDS. It
// converts every chunk once per 32 rows where the tiled kernel does once per
// 256, and needs neither barriers nor long runs of keys: a call too small to
// give every CU several of those tiles ends sooner with it.
//
// Bound: vector work. A step is 32 matrix operations of 16 passes and about
// 390 vector ones, 176 of them codes to halves; with 2000 tokens of 7B heads
// the vector pipes are busy 66% of the cycles, the matrix pipes 33% (that call
// is the tiled kernel's for this reason: 92 and 87 us). Small calls: 77 tokens
// of 3B heads 8.4 us, 512 of 7B heads 14.1, 16 x 77 22.3, 64 tokens at position
// 8000 33.8. On the way: every wave converting all 32 queries for itself cost
// 512 tokens 1.8 us more (a thread now converts an eighth of a row, once).
template <int HD, bool Q8>
struct Direct {
	static constexpr int EB = Q8 ? 1 : 2;
	static constexpr int KS = HD / 16, DT = HD / 32;
	static constexpr int KL = HD * EB / 32;   // 16-byte loads of a key per lane (a key is two lanes)
	static constexpr int VW = DT * EB / 4 > 0 ? DT * EB / 4 : 1;   // dwords of a value row per lane (DT dims; a row is 32 lanes)
	// The last step's lo halves stay in LDS where registers do not hold all (48 sequences over 6000 positions in 16 bits
	// 32.0 us, 33.8 with the compiler's choice in scratch memory).
	static constexpr bool kKeep = !Q8 && HD == 128;
	h8 qh[KS], ql[KS];
	float esc;
	f16v o[DT];
	float M, l;
	uint64_t big;   // as in Tile
	uint4 k[KL];
	uint32_t v[16][VW];
	float sc1;   // lanes 0..31: the keys' scales, 32..63: the values'

	// The rows' queries, times scale log2(e): a thread converts HD/8 dims of row tid/8 (src), once for all waves, and the
	// operands go through LDS (buf: HD * 128 bytes, es: 32 floats, both free again when this returns; keep: 1 KB that
	// stays). Step s of the score product takes dims 16 s + 8 h.. (halves) or 32 (s>>1) + 16 h + 8 (s&1).. (8 bits, as a
	// 16-byte load brings them) in lane half h.
	__device__ __forceinline__ void query(const float *src, float scale, uint8_t *buf, uint8_t *keep, float *es, int tid) {
		constexpr int N = HD / 8;
		const int t = tid & 7, row = tid >> 3, lane = tid & 63;
		float x[N], a = 0.0f;
#pragma unroll
		for (int j = 0; j < N; j += 4) {
			const float4 u = src ? *(const float4 *)(src + N * t + j) : make_float4(0, 0, 0, 0);
			x[j] = u.x * scale, x[j + 1] = u.y * scale, x[j + 2] = u.z * scale, x[j + 3] = u.w * scale;
		}
#pragma unroll
		for (int j = 0; j < N; j++) a = __builtin_fmaxf(a, __builtin_fabsf(x[j]));
		const int e = row_exp(max8(a));
		if (t == 0) es[row] = __builtin_ldexpf(1.0f, e);
#pragma unroll
		for (int j = 0; j < N / 8; j++) {
			const int m = N / 8 * t + j;   // dims 8 m..
			const int s = Q8 ? 2 * (m >> 2) + (m & 1) : m >> 1, h = Q8 ? (m >> 1) & 1 : m & 1;
			h8 hi, lo;
			split_q(x + 8 * j, e, hi, lo);
			*(h8 *)(buf + 16 * (128 * s + 32 * h + row)) = hi;
			*(h8 *)(buf + 16 * (128 * s + 64 + 32 * h + row)) = lo;
			if (kKeep && s == KS - 1) *(h8 *)(keep + 16 * (32 * h + row)) = lo;
		}
		__syncthreads();
#pragma unroll
		for (int s = 0; s < KS; s++) {
			qh[s] = *(const h8 *)(buf + 16 * (128 * s + lane));
			if (!kKeep || s < KS - 1) ql[s] = *(const h8 *)(buf + 16 * (128 * s + 64 + lane));
		}
		esc = es[lane & 31];
		__syncthreads();
#pragma unroll
		for (int d = 0; d < DT; d++)
#pragma unroll
			for (int v = 0; v < 16; v++) o[d][v] = 0.0f;
		M = kNone;
		l = 0.0f;
		big = 0;
	}

	// Tile row i is the key of row i in key_row's order (an involution): register v of a lane's scores is key
	// 16 (v>>3) + 8 h + (v&7).
	__device__ __forceinline__ void load_k(__amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t ksr, __amdgpu_buffer_rsrc_t vsr,
	                                       int key0, int lane) {
		const int i = lane & 31, h = lane >> 5;
		const uint32_t off = (uint32_t)(key0 + key_row(i)) * (HD * EB) + 16u * h;
#pragma unroll
		for (int n = 0; n < KL; n++) k[n] = ld_b128(kr, off + 32u * n);
		const uint32_t so = 4u * (uint32_t)(key0 + i);
		// (out of range loads are zeros: one of the two is)
		sc1 = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, ld_f32(ksr, h ? kBufNone : so)) |
		                                    __builtin_bit_cast(uint32_t, ld_f32(vsr, h ? so : kBufNone)));
	}
	// dims DT i..; keys 16 s + 8 h + j
	__device__ __forceinline__ void load_v(__amdgpu_buffer_rsrc_t vr, int key0, int lane) {
		const int i = lane & 31, h = lane >> 5;
#pragma unroll
		for (int n = 0; n < 16; n++) {
			const uint32_t off = ((uint32_t)(key0 + 16 * (n >> 3) + 8 * h + (n & 7)) * HD + DT * i) * EB;
			if (DT * EB == 2) v[n][0] = ld_b16(vr, off);
			if (DT * EB == 4) v[n][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, (int)off, 0, 0);
			if (DT * EB == 8) {
				const uint2 x = ld_b64(vr, off);
				v[n][0] = x.x;
				v[n][VW - 1] = x.y;
			}
		}
	}

	// As Stage's.
	__device__ __forceinline__ void keep(uint64_t written, int lane) {
		const int m = (int)((uint32_t)written >> (lane >> 5) * 8);
#pragma unroll
		for (int n = 0; n < 16; n++)
#pragma unroll
			for (int w = 0; w < VW; w++) v[n][w] &= (uint32_t)__builtin_amdgcn_sbfe(m, 16 * (n >> 3) + (n & 7), 1);
	}

	// The step's 32 keys from key0; mask: some row does not see all of them. sx: 128 floats of the wave's own in LDS, the
	// step's scales and every lane's base's e.
	__device__ __forceinline__ void scores(f16v &sc, const uint8_t *keep, int lane) {
#pragma unroll
		for (int v = 0; v < 16; v++) sc[v] = 0.0f;
#pragma unroll
		for (int s = 0; s < KS; s++) {
			h8 a;
			if (Q8) {
				const uint32_t w[4] = {k[(s >> 1) % KL].x, k[(s >> 1) % KL].y, k[(s >> 1) % KL].z, k[(s >> 1) % KL].w};
				const uint32_t x = w[2 * (s & 1)] ^ kFlip, y = w[2 * (s & 1) + 1] ^ kFlip;
				const h2 p = bytes_h2(x, kLo2), q2 = bytes_h2(x, kHi2), r = bytes_h2(y, kLo2), u = bytes_h2(y, kHi2);
				a = (h8){p.x, p.y, q2.x, q2.y, r.x, r.y, u.x, u.y};
			} else {
				a = __builtin_bit_cast(h8, k[s % KL]);
			}
			sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[s], sc, 0, 0, 0);
			sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, kKeep && s == KS - 1 ? *(const h8 *)(keep + 16 * lane) : ql[s], sc, 0, 0, 0);
		}
	}

	// The step's scales into sx; the exponent of the values' largest.
	__device__ __forceinline__ float scales(float *sx, int lane) {
		const float other = __shfl_xor(sc1, 32);
		const bool fin = __builtin_isfinite(lane < 32 ? other : sc1);   // the value row's scale
		const float e = scale_exp(wave_max(lane >= 32 && fin ? __builtin_fabsf(sc1) : 0.0f));
		// a value row that is not finite makes its score NaN
		sx[lane] = fin ? sc1 : (lane < 32 ? __builtin_nanf("") : 0.0f);
		__builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
		__builtin_amdgcn_wave_barrier();
		__builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
		return e;
	}

	template <class See>
	__device__ __forceinline__ void weigh(f16v &sc, float *sx, float e, bool mask, const See &see, int lane, h8 ph[2], h8 pl[2]) {
		const int h = lane >> 5;
		float mx = -INFINITY;
#pragma unroll
		for (int g = 0; g < 4; g++) {
			const float4 ks = *(const float4 *)(sx + 16 * (g >> 1) + 8 * h + 4 * (g & 1));
			const float kv[4] = {ks.x, ks.y, ks.z, ks.w};
#pragma unroll
			for (int j = 0; j < 4; j++) sc[4 * g + j] *= kv[j];
		}
		if (mask) {
			float vm = 0.0f;
#pragma unroll
			for (int g = 0; g < 4; g++) {
				const float4 vs = *(const float4 *)(sx + 32 + 16 * (g >> 1) + 8 * h + 4 * (g & 1));
				const float vv[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
				for (int j = 0; j < 4; j++) {
					const bool sees = see.sees(16 * (g >> 1) + 4 * (g & 1) + j);
					sc[4 * g + j] = sees ? sc[4 * g + j] : -INFINITY;
					vm = __builtin_fmaxf(vm, sees ? __builtin_fabsf(vv[j]) : 0.0f);
				}
			}
			e = scale_exp(__builtin_fmaxf(vm, __shfl_xor(vm, 32)));
		}
#pragma unroll
		for (int v = 0; v < 16; v++) mx = __builtin_fmaxf(mx, sc[v]);
		mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
		const float ue = __builtin_fmaf(mx, esc, e);
		float c = kUp - M;
		if (__ballot(passes(ue, M)) | big) {
			int f;
			if (__builtin_expect((__ballot(passes_big(ue, M)) | big) != 0, 0)) {
				Base at = {M, big ? sx[64 + lane] : 0.0f};
				f = move_up_any(at, mx * esc, e, ue);
				M = at.m;
				sx[64 + lane] = at.e;
				big = __ballot(at.big());
				big_scores<16>(sc, at, esc);
				c = at.big() ? 0.0f : kUp - M;
			} else {
				f = move_up(M, ue);
				c = kUp - M;
			}
			l = __builtin_ldexpf(l, f);
#pragma unroll
			for (int d = 0; d < DT; d++)
#pragma unroll
				for (int v = 0; v < 16; v++) o[d][v] = __builtin_ldexpf(o[d][v], f);
		}
#pragma unroll
		for (int g = 0; g < 4; g++) {
			const float4 vs = *(const float4 *)(sx + 32 + 16 * (g >> 1) + 8 * h + 4 * (g & 1));
			const float vv[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
			for (int j = 0; j < 4; j += 2) {
				const float p0 = exp2_(__builtin_fmaf(sc[4 * g + j], esc, c)), p1 = exp2_(__builtin_fmaf(sc[4 * g + j + 1], esc, c));
				l += p0;
				l += p1;
				h2 a, d;
				split2(p0 * vv[j], p1 * vv[j + 1], a, d);
				ph[g >> 1][4 * (g & 1) + j] = a.x;
				ph[g >> 1][4 * (g & 1) + j + 1] = a.y;
				pl[g >> 1][4 * (g & 1) + j] = d.x;
				pl[g >> 1][4 * (g & 1) + j + 1] = d.y;
			}
		}
	}

	// tile row i of dim tile d is dim DT i + d
	__device__ __forceinline__ void values(const h8 ph[2], const h8 pl[2]) {
#pragma unroll
		for (int s = 0; s < 2; s++)
#pragma unroll
			for (int d = 0; d < DT; d += 2) {
				h2 t[2][4];
#pragma unroll
				for (int p = 0; p < 4; p++) {
					const uint32_t a = v[8 * s + 2 * p][d * EB / 4], b = v[8 * s + 2 * p + 1][d * EB / 4];
					if (Q8) {
						const uint32_t m = __builtin_amdgcn_perm(b ^ kFlip, a ^ kFlip, d & 2 ? 0x07030602u : 0x05010400u);
						t[0][p] = bytes_h2(m, kLo2);
						t[1][p] = bytes_h2(m, kHi2);
					} else {
						t[0][p] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x05040100u));
						t[1][p] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x07060302u));
					}
				}
#pragma unroll
				for (int n = 0; n < 2; n++) {
					const h8 a = (h8){t[n][0].x, t[n][0].y, t[n][1].x, t[n][1].y, t[n][2].x, t[n][2].y, t[n][3].x, t[n][3].y};
					o[d + n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[s], o[d + n], 0, 0, 0);
					o[d + n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[s], o[d + n], 0, 0, 0);
				}
			}
	}
};

// The base and the sum that the waves' of a row meet at, and each wave's shift to it.
template <int R>
__device__ __forceinline__ Base meet(const float (&ml)[kWaves][R][4], int row, int x[kWaves], float &ls) {
	Base k[kWaves];
	float l[kWaves];
	bool big = false;
#pragma unroll
	for (int i = 0; i < kWaves; i++) {
		const float4 v = *(const float4 *)ml[i][row];
		k[i] = {v.x, v.y};
		l[i] = v.z;
		big |= v.y != 0.0f;
	}
	Base b = k[0];
#pragma unroll
	for (int i = 1; i < kWaves; i++) b.m = __builtin_fmaxf(b.m, k[i].m);
	if (__builtin_expect(big, 0)) {
		b = k[0];
#pragma unroll
		for (int i = 1; i < kWaves; i++) b = above(k[i], b) > 0.0f ? k[i] : b;
	}
	ls = 0.0f;
#pragma unroll
	for (int i = 0; i < kWaves; i++) {
		x[i] = steps_down(k[i], b);
		ls += __builtin_ldexpf(l[i], x[i]);
	}
	return b;
}

template <int HD>
struct DirectLds {
	alignas(16) float o[kWaves][32][HD + 4];
	alignas(16) float ml[kWaves][32][4];   // M, e and l
	alignas(16) float sx[kWaves][128];   // a wave's scales, and e of its rows' bases
	alignas(16) uint8_t keep[1024];
};

// Where rows go: row (token t, head g of the group) to o + t ot + g og, or to record first + t rt + g rg.
struct Dest {
	float *o;
	int64_t ot, og;
	Records rec;
	size_t first;
	int64_t rt, rg;
	__device__ __forceinline__ Dest(float *out, int64_t ldo, int HD) : o(out), ot(ldo), og(HD), rec{}, first(0), rt(0), rg(0) {}
	// (nrec to a query head, H heads to a token)
	__device__ __forceinline__ Dest(const Records &r, size_t f, int H, int nrec) : o(nullptr), ot(0), og(0), rec(r), first(f), rt((int64_t)H * nrec), rg(nrec) {}
};

// 32 rows over steps [c0, c1) of their tile's span. A lane's row: q (null: an idle row) and what it sees, tok << 4 | g its
// token and head (with kBlank: a row that sees nothing, whatever `row` says). (Places come from those two numbers after the
// steps: pointers held across them cost registers.)
constexpr int kBlank = 1 << 30;
template <int HD, bool Q8, class See>
__device__ __forceinline__ void direct_rows(const AttnKv &c, DirectLds<HD> &s, const Span &sp, int c0, int c1, const float *q,
                                            float scale, const See &seen, int tok_g, const Dest &dest) {
	constexpr int EB = Q8 ? 1 : 2;
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	Direct<HD, Q8> w;
	auto load_k = [&](int ch) {
		const size_t r = sp.first(ch) ? sp.r0 : sp.r1;
		const uint32_t n = (uint32_t)sp.top(ch);   // rows past it read as zeros
		w.load_k(stream_rsrc(uniform_ptr(c.k + r * HD * EB), n * HD * EB), stream_rsrc(uniform_ptr(c.ks + r), n * 4),
		         stream_rsrc(uniform_ptr(c.vs + r), n * 4), sp.key<32>(ch), fresh(lane));
	};
	auto load_v = [&](int ch) {
		const size_t r = sp.first(ch) ? sp.r0 : sp.r1;
		const uint32_t n = (uint32_t)sp.top(ch);
		w.load_v(stream_rsrc(uniform_ptr(c.v + r * HD * EB), n * HD * EB), sp.key<32>(ch), fresh(lane));
	};
	int ch = c0 + wave;
	if (ch < c1) {
		load_k(ch);
		load_v(ch);
	}
	__builtin_amdgcn_sched_barrier(0);
	// eight threads to a row, before the steps and after them (the row's pointers are in lane `row` of every wave)
	const int row = tid >> 3;
	auto from = [&](const void *p) {
		const uint64_t x = (uint64_t)(uintptr_t)p;
		return (uint64_t)(uint32_t)__shfl((int)(uint32_t)x, row) | ((uint64_t)(uint32_t)__shfl((int)(x >> 32), row) << 32);
	};
	w.query((const float *)(uintptr_t)from(q), scale, (uint8_t *)s.o, s.keep, s.sx[0], tid);
	const int lo = wave_min_i(tok_g >= 0 ? seen.lim : 0x7FFFFFFF), hi = seen.kHi ? wave_max_i(seen.lim) : 0;
	float *sx = s.sx[wave];
	for (; ch < c1; ch += kWaves) {
		const int key0 = sp.key<32>(ch), top = sp.top(ch);
		f16v sc;
		h8 ph[2], pl[2];
		w.scores(sc, s.keep, fresh(lane));
		if constexpr (See::kBlanks && !Q8)
			if (seen.template gaps<32>(key0)) w.keep(seen.written(key0), fresh(lane));
		const float e = w.scales(sx, lane);
		if (ch + kWaves < c1) load_k(ch + kWaves);
		__builtin_amdgcn_sched_barrier(0);
		See see = seen;
		see.at(key0 + 8 * (fresh(lane) >> 5), top, sp.first(ch));
		w.weigh(sc, sx, e, seen.template masks<32>(key0, top, sp.first(ch), lo, hi), see, fresh(lane), ph, pl);
		w.values(ph, pl);
		if (ch + kWaves < c1) load_v(ch + kWaves);
		__builtin_amdgcn_sched_barrier(0);
	}
	w.l += __shfl_xor(w.l, 32);
	// the waves' sums meet: row i, dims DT (8 (v>>2) + 4 h + (v&3)) + d
	const int at = fresh(tid), i = at & 31, h = (at >> 5) & 1, out = at >> 3;   // (out: this thread's row from here on)
#pragma unroll
	for (int v = 0; v < 16; v++) {
		float *to = &s.o[wave][i][w.DT * (8 * (v >> 2) + 4 * h + (v & 3))];
		if (w.DT == 4)
			*(float4 *)to = make_float4(w.o[0][v], w.o[1][v], w.o[2 % w.DT][v], w.o[3 % w.DT][v]);
		else
			*(float2 *)to = make_float2(w.o[0][v], w.o[1][v]);
	}
	if (h == 0) *(float4 *)s.ml[wave][i] = make_float4(w.M, w.big ? sx[64 + (at & 63)] : 0.0f, w.l, 0.0f);
	__syncthreads();
	const int tg = __shfl(tok_g, out);
	if (tg < 0) return;
	const bool blank = seen.kBlanks && tg & kBlank;
	if (blank && !dest.o) return;   // (nobody reads a record of nothing)
	const int tok = (seen.kBlanks ? tg & ~kBlank : tg) >> 4;
	const size_t r = dest.first + tok * dest.rt + (tg & 15) * dest.rg;
	float *to = dest.o ? dest.o + tok * dest.ot + (tg & 15) * dest.og : dest.rec.o + r * HD;
	int x[kWaves];
	float ls;
	const Base b = meet(s.ml, out, x, ls);
	if (blank) ls = 0.0f;
	const float z = !dest.o ? 1.0f : (ls == 0.0f ? 0.0f : 1.0f / ls);
#pragma unroll
	for (int d = 4 * (at & 7); d < HD; d += 32) {
		float4 a = make_float4(0, 0, 0, 0);
#pragma unroll
		for (int k = 0; k < kWaves; k++) {
			const float4 y = *(const float4 *)&s.o[k][out][d];
			a.x += __builtin_ldexpf(y.x, x[k]);
			a.y += __builtin_ldexpf(y.y, x[k]);
			a.z += __builtin_ldexpf(y.z, x[k]);
			a.w += __builtin_ldexpf(y.w, x[k]);
		}
		if (blank) a = make_float4(0, 0, 0, 0);
		*(float4 *)(to + d) = make_float4(a.x * z, a.y * z, a.z * z, a.w * z);
	}
	if (!dest.o && (at & 7) == 0) dest.rec.put(r, b, ls);
}

// What a prompt's row sees, lim its position and those before it.
template <bool WIN>
__device__ __forceinline__ auto row_sees(const AttnKv &c, int lim) {
	if constexpr (WIN) return Within{lim, c.window, 0};
	else return Below{lim};
}

template <int HD, bool Q8, bool WIN, int W>
__global__ __launch_bounds__(64 * W, 2) void prompt_kernel(AttnKv c, SeqTab t, ItemTab order, float *out, int64_t ldo, const float *q,
                                                        int64_t ldq, int G, float scale, Records rec) {
	__shared__ typename Tile<HD, Q8, W>::Lds s;
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	const int kvh = blockIdx.x % c.kvh;
	Item x;
	if (!item_of<kKeys, WIN>(t, &order, blockIdx.x / c.kvh, {c.prefix_len, c.window, c.sinks}, x)) return;
	const int r = 32 * wave + (lane & 31), tok = r / G, head = kvh * G + r - tok * G;
	const bool on = tok < x.ntok;
	const int lim = on ? t.start[x.sq] + x.tok0 + tok + 1 : 0;
	const int lo = wave_min_i(on ? lim : 0x7FFFFFFF), hi = wave_max_i(lim);
	const int64_t row = (int64_t)t.row[x.sq] + x.tok0 + tok;
	Tile<HD, Q8, W> w;
	w.chunks(c, span_of<kKeys, WIN>(c, kvh, x.slot, t.start[x.sq] + x.tok0, t.tile_tokens, x.end), x.c0, x.c1, row_sees<WIN>(c, lim), lo, hi,
	         s, tid, [&] { w.query(on ? q + row * ldq + head * HD : nullptr, scale, s, tid); });
	if (x.parts == 1) {
		w.put(on ? out + row * ldo + head * HD : nullptr, 1.0f / w.l, s, tid);
		return;
	}
	const size_t r0 = record_of(t, x, tok, c.kvh * G, head);
	w.put(on ? rec.o + r0 * HD : nullptr, 1.0f, s, tid);
	if (on && lane < 32) rec.put(r0, {w.M, w.big ? s.be[tid] : 0.0f}, w.l);
}

// The direct kernel's items: tiles of 32 rows, parts of `unit` steps of 32 keys.
template <int HD, bool Q8, bool WIN>
__global__ __launch_bounds__(64 * kWaves, 2) void prompt_direct_kernel(AttnKv c, SeqTab t, float *out, int64_t ldo, const float *q,
                                                               int64_t ldq, int G, float scale, Records rec) {
	__shared__ DirectLds<HD> s;
	const int lane = threadIdx.x & 63;
	const int kvh = blockIdx.x % c.kvh;
	Item x;
	if (!item_of<32, WIN>(t, nullptr, blockIdx.x / c.kvh, {c.prefix_len, c.window, c.sinks}, x)) return;
	const int r = lane & 31, tok = r / G, g = r - tok * G;
	const bool on = tok < x.ntok;
	const int64_t row = (int64_t)t.row[x.sq] + x.tok0;
	const int head = kvh * G, H = c.kvh * G;
	direct_rows<HD, Q8>(c, s, span_of<32, WIN>(c, kvh, x.slot, t.start[x.sq] + x.tok0, t.tile_tokens, x.end), x.c0, x.c1,
	                    on ? q + (row + tok) * ldq + (head + g) * HD : nullptr, scale,
	                    row_sees<WIN>(c, on ? t.start[x.sq] + x.tok0 + tok + 1 : 0), on ? tok << 4 | g : -1,
	                    x.parts == 1 ? Dest(out + row * ldo + head * HD, ldo, HD)
	                                 : Dest(rec, record_of(t, x, 0, H, head), H, t.nsplit[x.sq]));
}

// ── single tokens: the up to 16 query heads of a group over one sequence's own keys ──
//
// Workgroup (key/value head, sequence, part). Each wave takes steps of 32
// keys, codes straight from memory into the matrix-core operands
// (v_mfma_f32_16x16x32_f16: keys need no transposition, values are paired by
// byte permutes), the next ones on their way while these are used; the waves
// meet once, in LDS.
//
// Bound: memory behind a start of about 6 us (queries, first codes, the
// record, the join's launch): 16 sequences of 4096 positions read 69 MB in
// 19.1 us, 128 of 2000 270 MB in 52 us, 5.2 TB/s (a copy of 1 GiB runs at
// 5.1). One sequence of 1025 takes 9.3 us, the kernel 6.3 and the join 3.5. On
// the way: queries asked for before the first codes, and joins by one wave,
// 32768 and 20011 positions in 16 bits 20.8 us, then 17.9. The waves' number as
// a scalar, so that the loop is one for the compiler too: 64 sequences of 1000
// positions 15.1 us, now 14.8.
//
// Under a window the parts count the keys that are in sight, the sinks' in
// whole steps, then the window's from wherever it starts; no step before it is
// read, and its own start needs no mask. 64 sequences under 4096 keys, 236 MB:
// 44 us, 5.3 TB/s; one of 9001 under 1024: 6.4, and the join 3.6.
template <int HD, bool Q8>
struct Row16 {
	static constexpr int EB = Q8 ? 1 : 2;
	static constexpr int KS = HD / 32;                // 32-dim steps of the score product
	static constexpr int KL = HD * EB / 64;           // 16-byte loads of a key per lane (a key is four lanes)
	static constexpr int VD = HD / 16;                // dims per lane of a value row (a row is 16 lanes)
	static constexpr int VW = VD * EB / 4;            // dwords of them
	h8 qh[KS], ql[KS];
	float esc;
	f4 o[VD];
	float M, l;
	uint64_t big;   // as in Tile
	// a step's codes and scales
	struct Codes {
		uint4 k[2][KL];
		uint32_t v[8][VW];
		float ks[8], vs[8];
	};

	// dims of step s, lane group g, place j: KL loads of 16 bytes at 16 g + 64 i
	static __device__ __forceinline__ int dim0(int s, int g) {
		return Q8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
	}

	__device__ __forceinline__ void query(const float *q, float scale, int lane) {
		const int g = lane >> 4;
		float x[KS * 8], a = 0.0f;
#pragma unroll
		for (int s = 0; s < KS; s++) {
			float4 u = make_float4(0, 0, 0, 0), w = u;
			if (q) {
				u = *(const float4 *)(q + dim0(s, g));
				w = *(const float4 *)(q + dim0(s, g) + 4);
			}
			const float y[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
			for (int j = 0; j < 8; j++) {
				x[8 * s + j] = y[j] * scale;
				a = __builtin_fmaxf(a, __builtin_fabsf(x[8 * s + j]));
			}
		}
		a = __builtin_fmaxf(a, __shfl_xor(a, 16));
		a = __builtin_fmaxf(a, __shfl_xor(a, 32));
		const int e = row_exp(a);
		esc = __builtin_ldexpf(1.0f, e);
#pragma unroll
		for (int s = 0; s < KS; s++) split_q(x + 8 * s, e, qh[s], ql[s]);
#pragma unroll
		for (int d = 0; d < VD; d++) o[d] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
		M = kNone;
		l = 0.0f;
		big = 0;
	}

	// tile row i of key tile t is key 8 (i>>2) + 4 t + (i&3): a lane's eight scores are keys 8 g + 0..7
	static __device__ __forceinline__ void load_k(Codes &x, __amdgpu_buffer_rsrc_t kr, __amdgpu_buffer_rsrc_t ksr, int key0, int lane) {
		const int i = lane & 15, g = lane >> 4;
#pragma unroll
		for (int t = 0; t < 2; t++) {
			const uint32_t off = (uint32_t)(key0 + 8 * (i >> 2) + 4 * t + (i & 3)) * (HD * EB) + 16u * g;
#pragma unroll
			for (int n = 0; n < KL; n++) x.k[t][n] = ld_b128(kr, off + 64u * n);
		}
#pragma unroll
		for (int t = 0; t < 2; t++) {
			const float4 y = __builtin_bit_cast(float4, ld_b128(ksr, 4u * (uint32_t)(key0 + 8 * g + 4 * t)));
			x.ks[4 * t] = y.x, x.ks[4 * t + 1] = y.y, x.ks[4 * t + 2] = y.z, x.ks[4 * t + 3] = y.w;
		}
	}
	static __device__ __forceinline__ void load_v(Codes &x, __amdgpu_buffer_rsrc_t vr, __amdgpu_buffer_rsrc_t vsr, int key0, int lane) {
		const int i = lane & 15, g = lane >> 4;
#pragma unroll
		for (int j = 0; j < 8; j++) {
			const uint32_t off = ((uint32_t)(key0 + 8 * g + j) * HD + VD * i) * EB;
			if (VW == 1) x.v[j][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, (int)off, 0, 0);
			if (VW == 2) {
				const uint2 y = ld_b64(vr, off);
				x.v[j][0] = y.x;
				x.v[j][VW - 1] = y.y;
			}
			if (VW == 4) {
				const uint4 y = ld_b128(vr, off);
				x.v[j][0] = y.x;
				x.v[j][1 % VW] = y.y;
				x.v[j][2 % VW] = y.z;
				x.v[j][VW - 1] = y.w;
			}
		}
#pragma unroll
		for (int t = 0; t < 2; t++) {
			const float4 y = __builtin_bit_cast(float4, ld_b128(vsr, 4u * (uint32_t)(key0 + 8 * g + 4 * t)));
			x.vs[4 * t] = y.x, x.vs[4 * t + 1] = y.y, x.vs[4 * t + 2] = y.z, x.vs[4 * t + 3] = y.w;
		}
	}

	__device__ __forceinline__ void scores(const Codes &c, f4 sc[2]) {
#pragma unroll
		for (int t = 0; t < 2; t++) {
			sc[t] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
			for (int s = 0; s < KS; s++) {
				h8 a;
				if (Q8) {
					const uint4 &u4 = c.k[t][(s >> 1) % KL];
					const uint32_t w[4] = {u4.x, u4.y, u4.z, u4.w};
					const uint32_t x = w[2 * (s & 1)] ^ kFlip, y = w[2 * (s & 1) + 1] ^ kFlip;
					const h2 p = bytes_h2(x, kLo2), q2 = bytes_h2(x, kHi2), r = bytes_h2(y, kLo2), u = bytes_h2(y, kHi2);
					a = (h8){p.x, p.y, q2.x, q2.y, r.x, r.y, u.x, u.y};
				} else {
					a = __builtin_bit_cast(h8, c.k[t][s % KL]);
				}
				sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[s], sc[t], 0, 0, 0);
				sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[s], sc[t], 0, 0, 0);
			}
		}
	}

	// The exponent of the step's largest value scale. (Keys past the part read as zeros.) A value row that is not finite
	// makes its score NaN, through its key's scale.
	static __device__ __forceinline__ float exponent(Codes &cd) {
		float vm = 0.0f;
#pragma unroll
		for (int j = 0; j < 8; j++) {
			const bool fin = __builtin_isfinite(cd.vs[j]);
			cd.ks[j] = fin ? cd.ks[j] : __builtin_nanf("");
			cd.vs[j] = fin ? cd.vs[j] : 0.0f;
			vm = __builtin_fmaxf(vm, __builtin_fabsf(cd.vs[j]));
		}
		vm = __builtin_fmaxf(vm, __shfl_xor(vm, 16));
		return scale_exp(__builtin_fmaxf(vm, __shfl_xor(vm, 32)));
	}

	// Weights of the 32 keys from key0, those at end and past it left out.
	__device__ __forceinline__ void weigh(const Codes &cd, float *be, float e, f4 sc[2], int key0, int end, int lane, h8 &ph, h8 &pl) {
		const int g = lane >> 4;
		float x[8], mx = -INFINITY;
#pragma unroll
		for (int j = 0; j < 8; j++) {
			x[j] = key0 + 8 * g + j < end ? sc[j >> 2][j & 3] * cd.ks[j] : -INFINITY;
			mx = __builtin_fmaxf(mx, x[j]);
		}
		mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
		mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
		const float ue = __builtin_fmaf(mx, esc, e);
		float c = kUp - M;
		if (__ballot(passes(ue, M)) | big) {
			int f;
			if (__builtin_expect((__ballot(passes_big(ue, M)) | big) != 0, 0)) {
				Base at = {M, big ? be[threadIdx.x] : 0.0f};
				f = move_up_any(at, mx * esc, e, ue);
				M = at.m;
				be[threadIdx.x] = at.e;
				big = __ballot(at.big());
				big_scores<8>(x, at, esc);
				c = at.big() ? 0.0f : kUp - M;
			} else {
				f = move_up(M, ue);
				c = kUp - M;
			}
			l = __builtin_ldexpf(l, f);
#pragma unroll
			for (int d = 0; d < VD; d++)
#pragma unroll
				for (int v = 0; v < 4; v++) o[d][v] = __builtin_ldexpf(o[d][v], f);
		}
#pragma unroll
		for (int j = 0; j < 8; j += 2) {
			float w[2];
#pragma unroll
			for (int n = 0; n < 2; n++) {
				const float p = exp2_(__builtin_fmaf(x[j + n], esc, c));
				l += p;
				w[n] = p * cd.vs[j + n];
			}
			h2 a, b;
			split2(w[0], w[1], a, b);
			ph[j] = a.x, ph[j + 1] = a.y;
			pl[j] = b.x, pl[j + 1] = b.y;
		}
	}

	// tile row i of dim tile d is dim VD i + d
	__device__ __forceinline__ void values(const Codes &c, h8 ph, h8 pl) {
#pragma unroll
		for (int d = 0; d < VD; d += 2) {
			h2 t[2][4];
#pragma unroll
			for (int p = 0; p < 4; p++) {
				const uint32_t a = c.v[2 * p][d * EB / 4], b = c.v[2 * p + 1][d * EB / 4];
				if (Q8) {
					const uint32_t m = __builtin_amdgcn_perm(b ^ kFlip, a ^ kFlip, d & 2 ? 0x07030602u : 0x05010400u);
					t[0][p] = bytes_h2(m, kLo2);
					t[1][p] = bytes_h2(m, kHi2);
				} else {
					t[0][p] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x05040100u));
					t[1][p] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x07060302u));
				}
			}
#pragma unroll
			for (int n = 0; n < 2; n++) {
				const h8 a = (h8){t[n][0].x, t[n][0].y, t[n][1].x, t[n][1].y, t[n][2].x, t[n][2].y, t[n][3].x, t[n][3].y};
				o[d + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, o[d + n], 0, 0, 0);
				o[d + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[d + n], 0, 0, 0);
			}
		}
	}
};

// Keys per part of a sequence with n own keys in at most `parts` parts of `least` keys or more.
__device__ __forceinline__ int part_keys(int n, int parts, int least) {
	const int per = max((n + parts - 1) / parts, least);
	return (per + 32 * kWaves - 1) / (32 * kWaves) * (32 * kWaves);
}
// The part and sequence of a workgroup (of each key/value head), by its place
// (y, z) in a grid of own_grid, or the b-th in that order. A sequence's
// parts lie next to each other, on different CUs, while sequences are few.
// Where they fill the chip most parts are empty: all first parts come first,
// every next round shifted by one, so that the others go to all dies (64
// sequences of 1000 positions, one of 32000: 38 us, 85 with a sequence's parts
// together; but 8 of 1..8000 13.3 and 16.8).
dim3 own_grid(int kvh, int n_seq, int parts, int least) {
	return least < kLongPart ? dim3(kvh, parts, n_seq) : dim3(kvh, n_seq, parts);
}
__device__ __forceinline__ void part_of(int y, int z, int n_seq, int least, int &part, int &sq) {
	part = least < kLongPart ? y : z;
	sq = least < kLongPart ? z : (y + z) % n_seq;
}
__device__ __forceinline__ void part_of_nth(int b, int n_seq, int parts, int least, int &part, int &sq) {
	const int w = least < kLongPart ? parts : n_seq;
	part_of(b % w, b / w, n_seq, least, part, sq);
}
// A sequence's own keys [prefix, end): end, 0 where it has no slot.
__device__ __forceinline__ int own_end(const AttnKv &c, const int *slot, const int *len, int sq, int &sl) {
	sl = slot ? slot[sq] : sq;
	return sl < 0 || sl >= c.n_slots ? 0 : min(max(len[sq] + c.len_add, 0), c.max_seq);
}

// A sequence's own keys in the order that its parts take them: n of them, the first `sinks` (whole steps, if any) those
// from position 0, then those from b0 on.
struct Keys {
	int n, sinks, b0;
};
template <bool WIN>
__device__ __forceinline__ Keys own_keys(const AttnKv &c, int end) {
	if (!WIN) return {max(end - c.prefix_len, 0), 0, c.prefix_len};
	if (end - c.window <= c.sinks) return {end, 0, 0};
	const int s = (c.sinks + 31) / 32 * 32;
	return {s + c.window, s, end - c.window};
}

template <int HD>
struct DecodeLds {
	alignas(16) float o[kWaves][kMaxGroup][HD + 4];
	alignas(16) float ml[kWaves][kMaxGroup][4];   // M, e and l
	float be[64 * kWaves];   // e of the rows' bases
};

template <int HD, bool Q8, bool WIN>
__device__ __forceinline__ void decode_part(const AttnKv &c, DecodeLds<HD> &s, int kvh, int part, int sq, float *out, int64_t ldo,
                                            const float *q, int64_t ldq, const int *__restrict__ slot,
                                            const int *__restrict__ len, int G, float scale, int parts, int least, int rec0, int nrec,
                                            Records rec) {
	constexpr int EB = Q8 ? 1 : 2;
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
	int sl;
	const int end = own_end(c, slot, len, sq, sl);
	const Keys own = own_keys<WIN>(c, end);
	const int n = own.n, per = part_keys(n, parts, least);
	const int k0 = part * per, k1 = min(n, k0 + per);   // this part's keys
	if (k0 >= n && (part > 0 || nrec > 0)) return;   // a record that the join does not read
	const int first = own.b0 + k0, last = WIN ? end : min(end, first + per);   // (with a window: positions in at())
	const bool whole = nrec == 0 || (rec0 == 0 && n <= per);   // (the join leaves it alone)
	const int i = lane & 15, g = lane >> 4;
	const int head = kvh * G + i;
	// the first step's codes are on their way before the queries are asked for
	Row16<HD, Q8> w;
	const size_t r = ((size_t)(end > 0 ? sl : 0) * c.kvh + kvh) * c.max_seq;
	const uint32_t rows = (uint32_t)max(last, 0);
	auto kr = [&](uint32_t n) { return stream_rsrc(uniform_ptr(c.k + r * HD * EB), n * HD * EB); };
	auto vr = [&](uint32_t n) { return stream_rsrc(uniform_ptr(c.v + r * HD * EB), n * HD * EB); };
	auto ksr = [&](uint32_t n) { return stream_rsrc(uniform_ptr(c.ks + r), n * 4); };
	auto vsr = [&](uint32_t n) { return stream_rsrc(uniform_ptr(c.vs + r), n * 4); };
	// Codes on their way while others are used. 8 bits: two steps' in turn (64 sequences of 1000 positions 1.7 us less than
	// the other way). Halves, whose two steps would take 254 registers: the keys' of the next step once this one's
	// weights are formed, the values' after their products (32768 and 20011 positions 1.2 us less than in turn). (Keys from
	// `last` on read as zeros, from nowhere.)
	typename Row16<HD, Q8>::Codes ca, cb;
	// With a window key0 counts the part's keys in their order: at() is the position of the first of a step, top() that
	// past its last (a step past the part reads from nowhere).
	int key0 = WIN ? k0 + 32 * wave : first + 32 * wave;
	const int stop = WIN ? k1 : last;
	auto at = [&](int key) { return !WIN ? key : key >= k1 ? (int)rows : key < own.sinks ? key : own.b0 + (key - own.sinks); };
	auto top = [&](int key) { return WIN && key < own.sinks ? c.sinks : (int)rows; };
	auto load_k = [&](typename Row16<HD, Q8>::Codes &x, int key) { w.load_k(x, kr(top(key)), ksr(top(key)), at(key), lane); };
	auto load_v = [&](typename Row16<HD, Q8>::Codes &x, int key) { w.load_v(x, vr(top(key)), vsr(top(key)), at(key), lane); };
	auto load = [&](typename Row16<HD, Q8>::Codes &x, int key) {
		load_k(x, key);
		load_v(x, key);
		__builtin_amdgcn_sched_barrier(0);
	};
	auto step = [&](typename Row16<HD, Q8>::Codes &x) {
		f4 sc[2];
		h8 ph, pl;
		float e;
		if (Q8) e = w.exponent(x);
		w.scores(x, sc);
		if (!Q8) e = w.exponent(x);
		w.weigh(x, s.be, e, sc, at(key0), top(key0), lane, ph, pl);
		key0 += 32 * kWaves;
		if (!Q8) load_k(x, key0);
		w.values(x, ph, pl);
		if (!Q8) load_v(x, key0);
		if (Q8) __builtin_amdgcn_sched_barrier(0);
	};
	load(ca, key0);
	w.query(i < G ? q + sq * ldq + head * HD : nullptr, scale, lane);
	while (key0 < stop) {
		if (Q8) load(cb, key0 + 32 * kWaves);
		step(ca);
		if (!Q8) continue;
		if (key0 >= stop) break;
		load(ca, key0 + 32 * kWaves);
		step(cb);
	}
	w.l += __shfl_xor(w.l, 16);
	w.l += __shfl_xor(w.l, 32);
	// the waves' sums meet: rows i, dims VD (4 g + v) + d
#pragma unroll
	for (int v = 0; v < 4; v++)
#pragma unroll
		for (int d = 0; d < w.VD; d += 4)
			*(float4 *)&s.o[wave][i][w.VD * (4 * g + v) + d] =
			    make_float4(w.o[d][v], w.o[d + 1][v], w.o[d + 2][v], w.o[d + 3][v]);
	if (g == 0) *(float4 *)s.ml[wave][i] = make_float4(w.M, w.big ? s.be[tid] : 0.0f, w.l, 0.0f);
	__syncthreads();
	for (int t = tid; t < G * (HD / 4); t += 256) {
		const int row = t / (HD / 4), d = t % (HD / 4) * 4;
		int x[kWaves];
		float ls;
		const Base b = meet(s.ml, row, x, ls);
		float4 a = make_float4(0, 0, 0, 0);
#pragma unroll
		for (int k = 0; k < kWaves; k++) {
			const float4 y = *(const float4 *)&s.o[k][row][d];
			a.x += __builtin_ldexpf(y.x, x[k]);
			a.y += __builtin_ldexpf(y.y, x[k]);
			a.z += __builtin_ldexpf(y.z, x[k]);
			a.w += __builtin_ldexpf(y.w, x[k]);
		}
		const int hd = kvh * G + row;
		if (whole) {
			const float z = ls == 0.0f ? 0.0f : 1.0f / ls;
			*(float4 *)(out + sq * ldo + hd * HD + d) = make_float4(a.x * z, a.y * z, a.z * z, a.w * z);
		} else {
			const size_t r0 = ((size_t)sq * (c.kvh * G) + hd) * nrec + rec0 + part;
			*(float4 *)(rec.o + r0 * HD + d) = a;
			if (d == 0) rec.put(r0, b, ls);
		}
	}
}

template <int HD, bool Q8, bool WIN>
__global__ __launch_bounds__(256) void decode_kernel(AttnKv c, float *out, int64_t ldo, const float *q, int64_t ldq,
                                                     const int *__restrict__ slot, const int *__restrict__ len, int n_seq, int G,
                                                     float scale, int parts, int least, int nrec, Records rec) {
	__shared__ DecodeLds<HD> s;
	int part, sq;
	part_of(blockIdx.y, blockIdx.z, n_seq, least, part, sq);
	decode_part<HD, Q8, WIN>(c, s, blockIdx.x, part, sq, out, ldo, q, ldq, slot, len, G, scale, parts, least, 0, nrec, rec);
}

// A batch with a prefix in one launch, so that the two kinds of work fill each
// other's gaps: first the prefix's workgroups (rows are (sequence, head of the
// group), every row over the prefix's keys below its length), then the
// sequences' own; always to records.
template <int HD, bool Q8>
__global__ __launch_bounds__(64 * kWaves, 2) void prefix_kernel(AttnKv c, const float *q, int64_t ldq, const int *__restrict__ slot,
                                                        const int *__restrict__ len, int n_seq, int G, float scale,
                                                        int tiles, int pparts, int unit, int parts, int least, int nrec,
                                                        Records rec) {
	__shared__ union Lds {
		DirectLds<HD> a;
		DecodeLds<HD> b;
		__device__ Lds() {}
	} s;
	const int kvh = blockIdx.x % c.kvh;
	int b = blockIdx.x / c.kvh;
	if (b >= tiles * pparts) {
		b -= tiles * pparts;
		int own, sq;
		part_of_nth(b, n_seq, parts, least, own, sq);
		decode_part<HD, Q8, false>(c, s.b, kvh, own, sq, nullptr, 0, q, ldq, slot, len, G, scale, parts, least, pparts, nrec, rec);
		return;
	}
	const int lane = threadIdx.x & 63, part = b / tiles;
	const int64_t r = (int64_t)(b % tiles) * 32 + (lane & 31);
	const int sq = (int)(r / G), g = (int)(r - (int64_t)sq * G), head = kvh * G, H = c.kvh * G;
	const bool on = sq < n_seq;
	int lim = 0;
	if (on) {
		int sl;
		lim = min(own_end(c, slot, len, sq, sl), c.prefix_len);
	}
	const int nc = (c.prefix_len + 31) / 32;
	direct_rows<HD, Q8>(c, s.a, span_of<32, false>(c, kvh, c.prefix_slot, 0, 0, c.prefix_len), part * unit, min(nc, part * unit + unit),
	                    on ? q + (int64_t)sq * ldq + (head + g) * HD : nullptr, scale, Below{lim}, on ? sq << 4 | g : -1,
	                    Dest(rec, (size_t)head * nrec + part, H, nrec));
}

// a += y 2^f, ls += |l| 2^f
__device__ __forceinline__ void add_record(float4 &a, float &ls, float4 y, float l, int f) {
	ls += __builtin_ldexpf(__builtin_fabsf(l), f);
	a.x += __builtin_ldexpf(y.x, f);
	a.y += __builtin_ldexpf(y.y, f);
	a.z += __builtin_ldexpf(y.z, f);
	a.w += __builtin_ldexpf(y.w, f);
}

// One head's n records joined by a workgroup of kJoin waves: HD/4 lanes to a
// record (four dims each), so that 64 kJoin / (HD/4) of them are under way at
// a time; the lanes' sums meet by shuffles and then in LDS, in an order that n
// alone sets.
constexpr int kJoin = 4;
template <int HD>
__device__ __forceinline__ void join(const float *__restrict__ ro, const float2 *__restrict__ ml, const float *__restrict__ re, int n,
                                     float *dst) {
	constexpr int L = HD / 4, W = 64 * kJoin / L;
	__shared__ float m_s[kJoin], e_s[kJoin];
	__shared__ int big_s[kJoin];
	__shared__ float a_s[kJoin][HD + 4];
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	const int d = tid % L * 4, k0 = tid / L;
	// the first round's records and every thread's share of the maxima at once
	const int kf = max(min(k0, n - 1), 0);   // (there is room for a record where there is none)
	const float4 b0 = *(const float4 *)(ro + (size_t)kf * HD + d);
	const float2 x0 = ml[kf];
	// the largest base: the largest m, and where some have an e the most that a record is above that
	Base b = {kNone, 0.0f};
	bool some = false;
	for (int k = tid; k < n; k += 64 * kJoin) {
		const float2 x = ml[k];
		b.m = __builtin_fmaxf(b.m, x.x);
		some |= has_e(x);
	}
	b.m = wave_max(b.m);
	int big = __any(some);
	if (lane == 0) {
		m_s[wave] = b.m;
		big_s[wave] = big;
	}
	__syncthreads();
#pragma unroll
	for (int k = 0; k < kJoin; k++) {
		b.m = __builtin_fmaxf(b.m, m_s[k]);
		big |= big_s[k];
	}
	big = __builtin_amdgcn_readfirstlane(big);
	if (__builtin_expect(big, 0)) {
		float e = kNone;
		for (int k = tid; k < n; k += 64 * kJoin) e = __builtin_fmaxf(e, above(base_of(ml[k], re + k), b));
		e = wave_max(e);
		if (lane == 0) e_s[wave] = e;
		__syncthreads();
#pragma unroll
		for (int k = 0; k < kJoin; k++) e = __builtin_fmaxf(e, e_s[k]);
		b.e = e;
	}
	float ls = 0.0f;
	float4 a = make_float4(0, 0, 0, 0);
	if (__builtin_expect(big, 0)) {
		for (int k = k0; k < n; k += W) add_record(a, ls, *(const float4 *)(ro + (size_t)k * HD + d), ml[k].y, steps_down(base_of(ml[k], re + k), b));
	} else {
		if (k0 < n) add_record(a, ls, b0, x0.y, steps_down({x0.x, 0.0f}, b));
#pragma unroll 4
		for (int k = k0 + W; k < n; k += W) {
			const float2 x = ml[k];
			add_record(a, ls, *(const float4 *)(ro + (size_t)k * HD + d), x.y, steps_down({x.x, 0.0f}, b));
		}
	}
#pragma unroll
	for (int k = L; k < 64; k <<= 1) {
		ls += __shfl_xor(ls, k);
		a.x += __shfl_xor(a.x, k);
		a.y += __shfl_xor(a.y, k);
		a.z += __shfl_xor(a.z, k);
		a.w += __shfl_xor(a.w, k);
	}
	if (lane < L) {
		*(float4 *)&a_s[wave][d] = a;
		if (d == 0) a_s[wave][HD] = ls;
	}
	__syncthreads();
	if (tid < HD) {
		float o = a_s[0][tid], l = a_s[0][HD];
#pragma unroll
		for (int k = 1; k < kJoin; k++) {
			o += a_s[k][tid];
			l += a_s[k][HD];
		}
		dst[tid] = l == 0.0f ? 0.0f : o / l;
	}
}

template <int HD, bool WIN>
__global__ __launch_bounds__(64 * kJoin) void decode_join_kernel(AttnKv c, float *out, int64_t ldo, const int *__restrict__ slot,
                                                         const int *__restrict__ len, int H, int parts, int least, int rec0,
                                                         int nrec, const float *__restrict__ rec_o, const float2 *__restrict__ rec_ml,
                                                         const float *__restrict__ rec_e) {
	const int h = blockIdx.x, sq = blockIdx.y;
	int sl;
	const int n = own_keys<WIN>(c, own_end(c, slot, len, sq, sl)).n;
	const int per = part_keys(n, parts, least), used = n > 0 ? (n + per - 1) / per : 0;
	if (rec0 == 0 && used == 1) return;   // written at once
	const size_t rec = ((size_t)sq * H + h) * nrec;
	join<HD>(rec_o + rec * HD, rec_ml + rec, rec_e + rec, rec0 + used, out + sq * ldo + h * HD);
}

// n records, few, of one head joined for the four dims of ro.. (of each record HD floats).
__device__ __forceinline__ void join_few(const float *__restrict__ ro, int HD, const float2 *__restrict__ ml, const float *__restrict__ re,
                                         int n, float *dst) {
	// the first records and every maximum at once
	constexpr int P = 4;
	float4 y0[P];
	float2 x0[P];
#pragma unroll
	for (int k = 0; k < P; k++) {
		y0[k] = make_float4(0, 0, 0, 0);
		x0[k] = make_float2(kNone, 0.0f);
		if (k < n) {
			y0[k] = *(const float4 *)(ro + (size_t)k * HD);
			x0[k] = ml[k];
		}
	}
	Base b = {kNone, 0.0f};
	bool some = false;
#pragma unroll
	for (int k = 0; k < P; k++) {
		b.m = __builtin_fmaxf(b.m, x0[k].x);
		some |= has_e(x0[k]);
	}
	for (int k = P; k < n; k++) {
		const float2 x = ml[k];
		b.m = __builtin_fmaxf(b.m, x.x);
		some |= has_e(x);
	}
	const bool big = __any(some);
	if (__builtin_expect(big, 0)) {
		float e = kNone;
		for (int k = 0; k < n; k++) e = __builtin_fmaxf(e, above(base_of(ml[k], re + k), b));
		b.e = e;
	}
	float ls = 0.0f;
	float4 a = make_float4(0, 0, 0, 0);
	if (__builtin_expect(big, 0)) {
		for (int k = 0; k < n; k++) add_record(a, ls, *(const float4 *)(ro + (size_t)k * HD), ml[k].y, steps_down(base_of(ml[k], re + k), b));
	} else {
#pragma unroll
		for (int k = 0; k < P; k++)
			if (k < n) add_record(a, ls, y0[k], x0[k].y, steps_down({x0[k].x, 0.0f}, b));
#pragma unroll 4
		for (int k = P; k < n; k++) {
			const float4 y = *(const float4 *)(ro + (size_t)k * HD);
			const float2 x = ml[k];
			add_record(a, ls, y, x.y, steps_down({x.x, 0.0f}, b));
		}
	}
	const float z = ls == 0.0f ? 0.0f : 1.0f / ls;
	*(float4 *)dst = make_float4(a.x * z, a.y * z, a.z * z, a.w * z);
}

// The tokens whose tiles were split (the last ones of each sequence), few
// records each: HD/4 lanes to a query head, 1024/HD heads to a workgroup.
template <int HD, int K, bool WIN>
__global__ __launch_bounds__(256) void prompt_join_kernel(SeqTab t, Reach reach, float *out, int64_t ldo, int H,
                                                          const float *__restrict__ rec_o,
                                                          const float2 *__restrict__ rec_ml,
                                                          const float *__restrict__ rec_e) {
	constexpr int L = HD / 4;
	const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
	const int js = (int)(row / H), h = (int)(row - (int64_t)js * H), d = threadIdx.x % L * 4;
	if (js >= t.join[t.n]) return;
	int sq = 0;
	while (js >= t.join[sq + 1]) sq++;
	const int split = t.join[sq + 1] - t.join[sq];   // split tokens of the sequence
	const int j = js - t.join[sq], tok = t.len[sq] - split + j;
	const int tile = tok / t.tile_tokens, ns = t.nsplit[sq];
	const int nc = reach_steps<K, WIN>(reach, t.start[sq] + tile * t.tile_tokens, t.tile_tokens,
	                                   t.start[sq] + min((tile + 1) * t.tile_tokens, t.len[sq]));
	const int n = (nc + t.unit - 1) / t.unit;
	const size_t first = (size_t)t.rec[sq] + ((size_t)j * H + h) * ns;
	join_few(rec_o + first * HD + d, HD, rec_ml + first, rec_e + first, n, out + ((int64_t)t.row[sq] + tok) * ldo + (int64_t)h * HD + d);
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

AttnKv attn_kv(const hako_gpu_kv *kv, int prefix_slot, int prefix_len, int len_add) {
	return {(const uint8_t *)kv->k, (const uint8_t *)kv->v, kv->k_scale, kv->v_scale, kv->n_slots, kv->max_seq,
	        kv->n_kv_heads, prefix_slot, prefix_len, len_add, 0, 0};
}

// (a window or sinks past the cache's end are all of it)
AttnKv attn_kv_window(const hako_gpu_kv *kv, int len_add, int window, int sinks) {
	AttnKv c = attn_kv(kv, 0, 0, len_add);
	c.window = std::min(window, kv->max_seq);
	c.sinks = std::min(sinks, kv->max_seq);
	return c;
}

constexpr float kLog2e = 1.44269504088896340736f;

// Room for n records.
int records(size_t n, int HD, Records *r) {
	void *p = nullptr;
	if (int rc = workspace(kWsAttn, n * (HD + 3) * sizeof(float), &p)) return rc;
	r->o = (float *)p;
	r->ml = (float2 *)(r->o + n * HD);
	r->e = (float *)(r->ml + n);
	return HAKO_GPU_OK;
}

// How the single tokens of a batch are shared out: own keys (at most `own`) in up to `parts`
// parts of `least` keys or more, the prefix (tiles of 32 rows) in pparts parts
// of `unit` steps, nrec records to a query head (0: written at once).
struct DecodePlan {
	int64_t tiles;
	int parts, least, pparts, unit, nrec;
};
DecodePlan decode_plan(int own, int prefix_len, int kvh, int n_seq, int H, bool window) {
	DecodePlan p{};
	const int slots = 2 * cu_count();   // workgroups that run at once
	// own keys: parts of 32 keys a wave or more, until the workgroups fill the chip (16 sequences of 4096, 64 pairs of
	// sequence and head: 19.0 us with 8 parts, 18.5 with 4, 22.8 with 12). From a pair per CU on only long sequences are
	// split, for one among short ones (64 sequences, 256 pairs: one of 8000 and 63 of 100..400 positions 26 us, 63 in one
	// part; all of 4096 56 to 58 us, 50 to 53 in one part). The lengths are not known here, so the parts are those of
	// max_seq: 64 sequences of 1000 positions in slots of 2048 take 14.9 us, of 8192 17.4, of 32768 20.6
	const int64_t pairs = (int64_t)n_seq * kvh;
	// Windows of up to 8192 go undivided (64 sequences under 4096 49 us in parts of 2048, 44 in one; 128 under 2048 and some
	// sinks, whose step more makes a second part, 54 and 45). That is for batches of like lengths: of 63 sequences of
	// 100..400 positions and one of 8000 the long one is then a workgroup's alone (66.8 us under 8000, 38.3 under 4096, 22.2
	// under 2000; without a window, in parts, 26)
	p.least = pairs >= cu_count() ? (window ? kLongWindow : kLongPart) : 32 * kWaves;
	p.parts = (own + p.least - 1) / p.least;
	if (pairs < cu_count()) p.parts = std::min(p.parts, (int)(((prefix_len ? slots / 2 : slots) + pairs - 1) / pairs));
	p.parts = std::max(1, p.parts);
	// the prefix: parts of at least a step for each wave, until its tiles fill what the own keys leave, at least half the
	// chip (all of it / this: 48 sequences over 6000 positions 27.8 / 27.2 us, 8 over 16000 22.2 / 19.0, 32 of 3B heads
	// over 3000 20.0 / 15.3, 128 over 4000 42.4 / 39.3)
	p.tiles = ((int64_t)n_seq * (H / kvh) + 31) / 32;
	const int nc = (prefix_len + 31) / 32;
	p.unit = 1;
	if (nc) {
		const int64_t left = slots - std::min<int64_t>(slots / 2, pairs * p.parts);
		const int want = (int)std::max<int64_t>(1, left / (p.tiles * kvh));
		p.unit = std::max(kWaves, ((nc + want - 1) / want + kWaves - 1) / kWaves * kWaves);
		p.pparts = (nc + p.unit - 1) / p.unit;
	}
	p.nrec = p.pparts + p.parts > 1 ? p.pparts + p.parts : 0;
	return p;
}

// The most keys of its own that a sequence's token sees, a window's in whole steps after the sinks'.
int most_keys(const AttnKv &c) {
	return c.window ? (int)std::min<int64_t>(c.max_seq, ((int64_t)c.sinks + 31) / 32 * 32 + c.window) : c.max_seq - c.prefix_len;
}

template <int HD, bool Q8, bool WIN>
int decode(const AttnKv &c, float *out, int64_t ldo, const float *q, int64_t ldq, const int *slot, const int *len,
           int n_seq, int H, float scale) {
	const int G = H / c.kvh;
	const DecodePlan p = decode_plan(most_keys(c), c.prefix_len, c.kvh, n_seq, H, WIN);
	const int parts = p.parts, least = p.least, pparts = p.pparts, unit = p.unit, nrec = p.nrec;
	const int64_t tiles = p.tiles;
	Records rec{};
	if (nrec)
		if (int rc = records((size_t)n_seq * H * nrec, HD, &rec)) return rc;
	const int64_t blocks = (tiles * pparts + (int64_t)n_seq * parts) * c.kvh;
	if (blocks > kMaxThreads / (64 * kWaves)) return set_error(HAKO_GPU_EINVAL, "%lld workgroups in one call", (long long)blocks);
	if (!WIN && pparts) {
		hipLaunchKernelGGL((prefix_kernel<HD, Q8>), dim3((unsigned)blocks), dim3(64 * kWaves), 0, stream(), c, q, ldq, slot, len,
		                   n_seq, G, scale * kLog2e, (int)tiles, pparts, unit, parts, least, nrec, rec);
	} else {
		hipLaunchKernelGGL((decode_kernel<HD, Q8, WIN>), own_grid(c.kvh, n_seq, parts, least), dim3(256), 0, stream(), c, out, ldo, q, ldq, slot,
		                   len, n_seq, G, scale * kLog2e, parts, least, nrec, rec);
	}
	HK_LAUNCHED("attention");
	if (nrec) {
		hipLaunchKernelGGL((decode_join_kernel<HD, WIN>), dim3(H, n_seq), dim3(64 * kJoin), 0, stream(), c, out, ldo, slot, len, H, parts, least,
		                   pparts, nrec, rec.o, rec.ml, rec.e);
		HK_LAUNCHED("attention join");
	}
	return HAKO_GPU_OK;
}

// A launch's items in order of their length, so that the last ones to start
// are the shortest, where there are few enough for the table; their number,
// or 0.
template <int K, bool WIN>
int sort_items(const SeqTab &t, const Reach &reach, ItemTab &order) {
	struct Len {
		int steps;
		uint32_t item;
	} len[kItems];
	int n = 0;
	order.n = 0;
	for (int s = 0; s < t.n; s++) {
		const int tiles = (t.len[s] + t.tile_tokens - 1) / t.tile_tokens;
		if (tiles > kItems || t.nsplit[s] > 256) return 0;
		for (int i = tiles - 1; i >= 0; i--) {
			const int nc = reach_steps<K, WIN>(reach, t.start[s] + i * t.tile_tokens, t.tile_tokens,
			                                   t.start[s] + std::min((i + 1) * t.tile_tokens, t.len[s]));
			const int parts = (nc + t.unit - 1) / t.unit, per = (nc + parts - 1) / parts;
			if (n + parts > kItems) return 0;
			for (int k = 0; k < parts; k++) len[n++] = {std::min(per, nc - k * per), (uint32_t)s << 26 | (uint32_t)(i << 8 | k)};
		}
	}
	std::sort(len, len + n, [](const Len &a, const Len &b) { return a.steps != b.steps ? a.steps > b.steps : a.item < b.item; });
	for (int i = 0; i < n; i++) order.item[i] = len[i].item;
	return order.n = n;
}

// One launch of up to kSeqs sequences, in the order given (the longest
// first): tiles of `rows` query rows, steps of K keys, parts of `unit` steps.
template <int HD, bool Q8, int K, bool WIN, class Launch>
int prompt_launch(const AttnKv &c, const Reach &reach, SeqTab &t, float *out, int64_t ldo, int H, int rows, int64_t unit, Launch launch) {
	t.tile_tokens = rows / (H / c.kvh);
	t.unit = (int)std::min<int64_t>(unit, 0x7FFFFFFF);
	int64_t items = 0, recs = 0;
	for (int s = 0; s < t.n; s++) {
		const int tiles = (t.len[s] + t.tile_tokens - 1) / t.tile_tokens;
		auto steps = [&](int tile) {
			return reach_steps<K, WIN>(reach, t.start[s] + tile * t.tile_tokens, t.tile_tokens,
			                           (int)(t.start[s] + std::min<int64_t>((int64_t)(tile + 1) * t.tile_tokens, t.len[s])));
		};
		t.nsplit[s] = (steps(tiles - 1) + t.unit - 1) / t.unit;
		t.item[s] = (int)items;
		items += (int64_t)tiles * t.nsplit[s];
		t.rec[s] = (uint32_t)recs;
		// the first tile of more than `unit` steps (a tile sees no fewer than those before it)
		int lo = 0, hi = tiles;
		while (lo < hi) {
			const int mid = (lo + hi) / 2;
			if (steps(mid) <= t.unit) lo = mid + 1;
			else hi = mid;
		}
		const int first = (int)std::min<int64_t>((int64_t)lo * t.tile_tokens, t.len[s]);
		t.join[s + 1] = t.join[s] + t.len[s] - first;
		recs += (int64_t)(t.len[s] - first) * H * t.nsplit[s];
	}
	t.item[t.n] = (int)items;
	if (items * c.kvh > kMaxThreads / 512 || recs > 0xFFFFFFFFll || (int64_t)t.join[t.n] * H * (HD / 4) > kMaxThreads)
		return set_error(HAKO_GPU_EINVAL, "%lld tiles and %lld records in one call", (long long)(items * c.kvh), (long long)recs);
	Records rec{};
	if (recs)
		if (int rc = records((size_t)recs, HD, &rec)) return rc;
	launch(items, rec);
	HK_LAUNCHED("attention");
	if (recs) {
		const int64_t blocks = ((int64_t)t.join[t.n] * H * (HD / 4) + 255) / 256;
		hipLaunchKernelGGL((prompt_join_kernel<HD, K, WIN>), dim3((unsigned)blocks), dim3(256), 0, stream(), t, reach, out, ldo, H, rec.o, rec.ml, rec.e);
		HK_LAUNCHED("attention join");
	}
	return HAKO_GPU_OK;
}

// Steps of K keys over all tiles of `tokens` tokens: a sequence's tiles at the
// mean of its first and last one's; with a window the tiles that still see
// everything so, the others at the last one's.
template <int K, bool WIN>
int64_t all_steps(const AttnKv &c, const Reach &reach, const SeqTab &t, int tokens) {
	int64_t n = 0;
	for (int s = 0; s < t.n; s++) {
		const int64_t tiles = (t.len[s] + tokens - 1) / tokens;
		auto steps = [&](int64_t tile) {
			const int first = (int)(t.start[s] + tile * tokens);
			return (int64_t)reach_steps<K, WIN>(reach, first, tokens, std::min(first + tokens, t.start[s] + t.len[s]));
		};
		int64_t grow = tiles;
		if (WIN) {   // tiles with start + (tile + 1) tokens - window <= sinks
			const int64_t room = (int64_t)reach.sinks + reach.window - t.start[s];
			grow = std::min(tiles, room < 0 ? 0 : room / tokens);
		}
		if (grow) n += (grow * (steps(0) + steps(grow - 1)) + 1) / 2;
		n += (tiles - grow) * steps(tiles - 1);
	}
	return n * c.kvh;
}

// The tiles of `tokens` tokens of a launch, with their key/value heads, and the steps of the longest.
struct Tiles {
	int64_t items, most;
};
template <int K, bool WIN>
Tiles tiles_of(const AttnKv &c, const Reach &reach, const SeqTab &t, int tokens) {
	Tiles x{};
	for (int s = 0; s < t.n; s++) {
		const int64_t n = (t.len[s] + tokens - 1) / tokens;
		const int first = (int)(t.start[s] + (n - 1) * tokens);
		x.items += n * c.kvh;
		x.most = std::max<int64_t>(x.most, reach_steps<K, WIN>(reach, first, tokens, t.start[s] + t.len[s]));
	}
	return x;
}

// The tiled kernel of W waves; as many workgroups run at once as fill a CU with eight.
template <int HD, bool Q8, bool WIN, int W>
int prompt_tiled(const AttnKv &c, const Reach &reach, SeqTab &t, float *out, int64_t ldo, const float *q, int64_t ldq, int H, float scale) {
	const int G = H / c.kvh;
	const int64_t slots = 8 / W * cu_count(), all = all_steps<kKeys, WIN>(c, reach, t, 32 * W / G);
	int64_t unit = (3 * all + 2 * slots - 1) / (2 * slots);
	if (WIN) {
		// tiles under a window are much alike: as many parts as the chip takes at once, and none where half a share is in
		// question (1500 tokens under 512, two thirds of the chip: 62 us in two parts, 43 in one)
		const Tiles x = tiles_of<kKeys, WIN>(c, reach, t, 32 * W / G);
		const int64_t parts = x.items ? slots / x.items : 0;
		unit = parts > 1 ? (x.most + parts - 1) / parts : 2 * ((all + slots - 1) / slots);
	}
	return prompt_launch<HD, Q8, kKeys, WIN>(
	    c, reach, t, out, ldo, H, 32 * W, std::max<int64_t>(4, unit),
	    [&](int64_t items, const Records &rec) {
		    ItemTab order;
		    if (const int n = sort_items<kKeys, WIN>(t, reach, order)) items = n;
		    hipLaunchKernelGGL((prompt_kernel<HD, Q8, WIN, W>), dim3((unsigned)(items * c.kvh)), dim3(64 * W), 0, stream(), c, t, order, out,
		                       ldo, q, ldq, G, scale * kLog2e, rec);
	    });
}

// Which kernel under a window, 1 the direct one, 2 or 3 the tiled one of eight or four waves: the least of their times by
// a model of a start, rounds of items and steps. Its constants, in us, are fits to heads of 128 / 64 on one MI355X: an
// item takes 9 / 4.2 and 1.35 / 1 a step of a wave (16 bits and 128: 1.6) in the direct kernel, 13 / 8.5 and 2.8 / 1.85 a
// chunk in the tiled one, where tiles of four waves, two at a time on a CU, cost (0.96 + 0.0065 chunks) times as much for
// the same rows but end in half rounds. Model / measured for 7B heads, 8 bits, by the three: 512 tokens at 3000 under 512
// 20 30 - / 20 36 33; 2000 under 512 63 46 - / 58 44 52; 4096 under 256 100 65 60 / 90 67 66; 8192 under 2048 576 440 510
// / 573 416 436.
template <int HD, bool Q8>
int window_kernel(const AttnKv &c, const Reach &reach, const SeqTab &t, int G) {
	const double cu = cu_count(), slots = 2 * cu, start = 5.0, join = 4.0;
	const double di = HD == 128 ? 9.0 : 4.2, ds = HD == 64 ? 1.0 : Q8 ? 1.35 : 1.6, ti = HD == 128 ? 13.0 : 8.5, ts = HD == 128 ? 2.8 : 1.85;
	const Tiles d = tiles_of<32, true>(c, reach, t, 32 / G), x = tiles_of<kKeys, true>(c, reach, t, 256 / G);
	const double dn = (double)d.items, n = (double)x.items, all = (double)all_steps<kKeys, true>(c, reach, t, 256 / G);
	double direct, tiled, small = 1e30;
	if (dn >= slots) {
		direct = start + (dn * di + ds * (double)all_steps<32, true>(c, reach, t, 32 / G) / kWaves) / slots;
	} else {
		const double parts = std::max(1.0, floor(slots / dn));
		direct = start + di + ds * ceil(d.most / (kWaves * parts)) + (parts > 1 ? join : 0.0);
	}
	if (n > cu) {
		const double item = ti + ts * all / n, r = n / cu, part = r - floor(r);
		tiled = start + ceil(r) * item;
		small = start + (floor(r) + (part > 0.0 ? std::max(part, 0.5) : 0.0)) * (0.96 + 0.0065 * all / n) * item;
	} else {
		const double parts = std::max(1.0, floor(cu / n));
		tiled = start + ti + ts * ceil(x.most / parts) + (parts > 1 ? join : 0.0);
	}
	return direct <= std::min(tiled, small) ? 1 : tiled <= small ? 2 : 3;
}

// Which kernel (one MI355X, heads of 128, us by the direct / the tiled one):
//   tokens        wave-steps (32 rows x 32 keys)   8 bits        16 bits
//   7B heads  200       0.8 thousand               9.3 / 20.5    9.9 / 20.5
//            1000      16.5                       33.6 / 41.2   37.5 / 41.2
//             512 at 3000   52                    70.6 / 72.8   79.6 / 73.6
//            2000      64                         92.0 / 87.2    109 / 88.5
//            3000     143                          187 / 153     221 / 156
//   3B heads 2000      32                         52.7 / 59.9   58.6 / 60.4
//            3000      71                         98.7 / 103     116 / 105
//             512 at 3000   26                    59.8 / 51.4   73.0 / 51.7
// So the direct one up to 55 wave-steps for each SIMD. (One query group of 16
// goes as 3B heads, heads of 64 cross at about the same work. Some hundred
// tokens far on in a slot of few heads are better off with the tiled one, the
// last row; the rule does not see that.)
//
// Parts: the tiled kernel splits tiles of more than 1.5 times an equal share
// of the work (1, 1.5, 2 times: packed prompts of 4097 tokens 109 / 100 / 106
// us, 2 x 1500 tokens 98 / 83 / 83: a part costs its record's way to memory and
// back); the direct one tiles of more than a share where they are too few for
// the chip (64 tokens at position 8000: 34 us, 37 at two shares), else of more
// than two (512 at 3000: 70, 115 at one).
template <int HD, bool Q8, bool WIN>
int prompt(const AttnKv &c, SeqTab &t, float *out, int64_t ldo, const float *q, int64_t ldq, int H, float scale) {
	const int G = H / c.kvh;
	const int64_t cu = cu_count(), slots = 2 * cu;   // workgroups of the direct kernel that run at once
	const Reach reach = {c.prefix_len, c.window, c.sinks};
	const int64_t steps = all_steps<32, WIN>(c, reach, t, 32 / G);
	const int kernel = g_attn_prompt ? g_attn_prompt : WIN ? window_kernel<HD, Q8>(c, reach, t, G) : steps > 55 * 4 * cu ? 2 : 1;
	if (WIN && kernel == 3) return prompt_tiled<HD, Q8, WIN, WIN ? 4 : 8>(c, reach, t, out, ldo, q, ldq, H, scale);
	if (kernel != 1) return prompt_tiled<HD, Q8, WIN, 8>(c, reach, t, out, ldo, q, ldq, H, scale);
	int64_t tiles = 0;
	for (int s = 0; s < t.n; s++) tiles += (t.len[s] + 32 / G - 1) / (32 / G);
	const int64_t share = (steps + slots - 1) / slots;
	return prompt_launch<HD, Q8, 32, WIN>(c, reach, t, out, ldo, H, 32,
	                                      std::max<int64_t>(4 * kWaves, 2 * tiles * c.kvh <= slots ? share : 2 * share),
	                                      [&](int64_t items, const Records &rec) {
		                                      hipLaunchKernelGGL((prompt_direct_kernel<HD, Q8, WIN>), dim3((unsigned)(items * c.kvh)),
		                                                         dim3(64 * kWaves), 0, stream(), c, t, out, ldo, q, ldq, G, scale * kLog2e, rec);
	                                      });
}

// ── drafted trees ──
//
// Rows are (node, head of the group) of one sequence, node-major, against the
// sequence's text and the tree's own rows behind it. A row sees all of the text
// and of the 64 keys from base on its mask's bits: a step's 32 or 64 bits are
// one shift of the mask (Nodes::at), so that masked steps cost what a causal
// mask's do and the others nothing. Nodes that are not there have mask 0; their
// waves pass no chunk and their rows have no records. Their cache rows may never
// have been written: halves there are taken as zeros (Stage::keep; 0.2 us of one
// tree of 26, 1.2 of 34 for 8 of 64 at 1000 in 16 bits).
//
// Two kernels as for prompts. 32-row tiles straight from memory (direct): small
// trees, latency. One tree of 26 nodes at 1025, 3B heads: 8.4 us, most
// of it places, masks, first codes and queries one after the other; the join
// 3.6. Tiles of 256 or 128 rows (tiled): 16 trees of 64 nodes at 4096, 7B
// heads, 120 GFLOP with both halves: 119 to 133 us by the chip, and the join
// 9.4 (11 before it asked for its first records with their bases); tiles of 512
// rows for 448, and parts of 33 chunks behind a start of 13 us, are what is
// lost. 32 trees of 1..16 nodes over a prefix of 3001 in 16 bits: 62 us and 6,
// tiles half full.

// Where a sequence's nodes go: rows [base, end), base 0 and no rows where it has no place.
__device__ __forceinline__ bool tree_place(const AttnKv &c, const int *slot, const int *base, int sq, int N, int &sl, int &b, int &end) {
	sl = slot ? slot[sq] : sq;
	b = base[sq];
	const bool on = sl >= 0 && sl < c.n_slots && b >= 0;
	sl = on ? sl : 0;
	b = on ? min(b, c.max_seq) : 0;
	end = on ? min(b + N, c.max_seq) : 0;
	return on;
}
// The nodes of a row that it sees, 0: it is not there.
__device__ __forceinline__ uint64_t tree_bits(const uint64_t *seen, int64_t row, int N) {
	return N < 64 ? seen[row] & ((1ull << N) - 1) : seen[row];
}
// The nodes that some row of the sequence sees. (Only halves need them: see Stage::keep.)
template <bool Q8>
__device__ __forceinline__ uint64_t tree_any(const uint64_t *seen, int sq, int N, int lane) {
	return Q8 ? 0 : wave_or(lane < N ? seen[(int64_t)sq * N + lane] : 0);
}
// Steps per part of a tile with nc steps, in whole rounds of R.
template <int R>
__device__ __forceinline__ int tree_part(int nc, int parts) {
	return max(((nc + parts - 1) / parts + R - 1) / R * R, R);
}

// A workgroup's key/value head, sequence, part and tile. Workgroups go to the eight dies in turn: the tiles of a part,
// which read the same keys, follow one another on one die.
__device__ __forceinline__ bool tree_item(int n_kvh, int n_seq, int parts, int tiles, int &kvh, int &sq, int &part, int &tile) {
	const int g = blockIdx.x / (8 * tiles), r = blockIdx.x - g * (8 * tiles);
	const int p = 8 * g + r % 8;   // (part, sequence, head)
	tile = r / 8;
	kvh = p % n_kvh;
	sq = p / n_kvh % n_seq;
	part = p / n_kvh / n_seq;
	return part < parts;
}
unsigned tree_blocks(int64_t items, int64_t tiles) { return (unsigned)((items + 7) / 8 * 8 * tiles); }

// Zeros for the 32 rows (node, g) that a wave's lanes hold (node -1: none), by a workgroup whose waves hold the same.
template <int HD>
__device__ __forceinline__ void tree_blank(int node, int g, float *out, int64_t ldo) {
	const int row = threadIdx.x >> 3, n = __shfl(node, row), hd = __shfl(g, row);
	if (n < 0) return;
#pragma unroll
	for (int d = 4 * (threadIdx.x & 7); d < HD; d += 32) *(float4 *)(out + n * ldo + hd * HD + d) = make_float4(0, 0, 0, 0);
}

template <int HD, bool Q8>
__global__ __launch_bounds__(64 * kWaves, 2) void tree_kernel(AttnKv c, float *out, int64_t ldo, const float *q, int64_t ldq,
                                                              const int *__restrict__ slot, const int *__restrict__ base,
                                                              const uint64_t *__restrict__ seen, int n_seq, int N, int G, float scale,
                                                              int parts, Records rec) {
	__shared__ DirectLds<HD> s;
	int kvh, sq, part, tile;
	if (!tree_item(c.kvh, n_seq, parts, (N * G + 31) / 32, kvh, sq, part, tile)) return;
	const int lane = threadIdx.x & 63, r = 32 * tile + (lane & 31), node = r / G, g = r - node * G;
	const int head = kvh * G, H = c.kvh * G;
	const bool on = node < N;
	const int64_t row = (int64_t)sq * N + node;
	uint64_t bits = on ? tree_bits(seen, row, N) : 0;   // (asked for together with the place)
	const uint64_t any = tree_any<Q8>(seen, sq, N, lane);
	int sl, b, end;
	if (!tree_place(c, slot, base, sq, N, sl, b, end)) bits = 0;
	const Span sp = span_of<32, false>(c, kvh, sl, 0, 0, end);
	const int nc = sp.n0 + (max(end - sp.b0, 0) + 31) / 32;
	const int per = tree_part<kWaves>(nc, parts), c0 = part * per;
	if (c0 >= nc && part > 0) return;   // a record that the join does not read
	if (!__any(bits != 0)) {   // nodes that are not there, as in the last tiles of a padded tree
		if (parts == 1) tree_blank<HD>(on ? node : -1, g, out + (int64_t)sq * N * ldo + head * HD, ldo);
		return;
	}
	direct_rows<HD, Q8>(c, s, sp, c0, min(nc, c0 + per), on && bits ? q + row * ldq + (head + g) * HD : nullptr, scale, Nodes{b, bits, any, 0},
	                    on ? node << 4 | g | (bits ? 0 : kBlank) : -1,
	                    parts == 1 ? Dest(out + (int64_t)sq * N * ldo + head * HD, ldo, HD)
	                               : Dest(rec, ((size_t)sq * N * H + head) * parts + part, H, parts));
}

// The same by the tiled kernel, tiles of 32 W rows.
template <int HD, bool Q8, int W>
__global__ __launch_bounds__(64 * W, 2) void tree_tiled_kernel(AttnKv c, float *out, int64_t ldo, const float *q, int64_t ldq,
                                                               const int *__restrict__ slot, const int *__restrict__ base,
                                                               const uint64_t *__restrict__ seen, int n_seq, int N, int G, float scale,
                                                               int parts, Records rec) {
	__shared__ typename Tile<HD, Q8, W>::Lds s;
	int kvh, sq, part, tile;
	if (!tree_item(c.kvh, n_seq, parts, (N * G + 32 * W - 1) / (32 * W), kvh, sq, part, tile)) return;
	const int tid = threadIdx.x, lane = tid & 63, r = 32 * (W * tile + (tid >> 6)) + (lane & 31), node = r / G, g = r - node * G;
	const int head = kvh * G + g, H = c.kvh * G;
	const bool on = node < N;
	const int64_t row = (int64_t)sq * N + node;
	uint64_t bits = on ? tree_bits(seen, row, N) : 0;
	const uint64_t any = tree_any<Q8>(seen, sq, N, lane);
	int sl, b, end;
	if (!tree_place(c, slot, base, sq, N, sl, b, end)) bits = 0;
	const Span sp = span_of<kKeys, false>(c, kvh, sl, 0, 0, end);
	const int nc = sp.n0 + (max(end - sp.b0, 0) + kKeys - 1) / kKeys;
	const int per = tree_part<1>(nc, parts), c0 = part * per;
	if (c0 >= nc && part > 0) return;   // a record that the join does not read
	// a wave without nodes sees nothing, a workgroup without any passes no chunk
	const int hi = __any(bits != 0) ? end : 0, stop = __syncthreads_or(hi) ? min(nc, c0 + per) : c0;
	Tile<HD, Q8, W> w;
	w.chunks(c, sp, c0, stop, Nodes{b, bits, any, 0}, b, hi, s, tid,
	         [&] { w.query(on ? q + row * ldq + head * HD : nullptr, scale, s, tid); });
	if (parts == 1) {
		if (!bits) w.clear();
		w.put(on ? out + row * ldo + head * HD : nullptr, w.l == 0.0f ? 0.0f : 1.0f / w.l, s, tid);
		return;
	}
	const size_t r0 = ((size_t)row * H + head) * parts + part;
	w.put(bits ? rec.o + r0 * HD : nullptr, 1.0f, s, tid);
	if (bits && lane < 32) rec.put(r0, {w.M, w.big ? s.be[tid] : 0.0f}, w.l);
}

// A sequence's records, as many as its text has parts, joined; zeros for nodes that are not there.
template <int HD, int K, int R>
__global__ __launch_bounds__(256) void tree_join_kernel(AttnKv c, float *out, int64_t ldo, const int *__restrict__ slot,
                                                        const int *__restrict__ base, const uint64_t *__restrict__ seen,
                                                        int n_seq, int N, int H, int parts, const float *__restrict__ rec_o, const float2 *__restrict__ rec_ml,
                                                        const float *__restrict__ rec_e) {
	constexpr int L = HD / 4;
	const int64_t i = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
	const int64_t row = i / H;
	const int h = (int)(i - row * H), d = threadIdx.x % L * 4, sq = (int)(row / N);
	if (sq >= n_seq) return;
	int sl, b, end;
	float *to = out + row * ldo + (int64_t)h * HD + d;
	const uint64_t bits = tree_bits(seen, row, N);
	if (!tree_place(c, slot, base, sq, N, sl, b, end) || !bits) {
		*(float4 *)to = make_float4(0, 0, 0, 0);
		return;
	}
	const int nc = tile_steps<K>(end, c.prefix_len), per = tree_part<R>(nc, parts);
	const size_t first = (size_t)i * parts;
	join_few(rec_o + first * HD + d, HD, rec_ml + first, rec_e + first, max((nc + per - 1) / per, 1), to);
}

// The same for many parts: a workgroup a row and head.
template <int HD, int K, int R>
__global__ __launch_bounds__(64 * kJoin) void tree_join_wide_kernel(AttnKv c, float *out, int64_t ldo, const int *__restrict__ slot,
                                                                    const int *__restrict__ base, const uint64_t *__restrict__ seen,
                                                                    int N, int parts, const float *__restrict__ rec_o,
                                                                    const float2 *__restrict__ rec_ml, const float *__restrict__ rec_e) {
	const int h = blockIdx.x, row = blockIdx.y;
	int sl, b, end;
	const uint64_t bits = tree_bits(seen, row, N);
	if (!tree_place(c, slot, base, row / N, N, sl, b, end) || !bits) {
		if (threadIdx.x < HD) out[row * ldo + h * HD + threadIdx.x] = 0.0f;
		return;
	}
	const int nc = tile_steps<K>(end, c.prefix_len), per = tree_part<R>(nc, parts);
	const size_t first = ((size_t)row * gridDim.x + h) * parts;
	join<HD>(rec_o + first * HD, rec_ml + first, rec_e + first, max((nc + per - 1) / per, 1), out + row * ldo + h * HD);
}

// Trees of N nodes over parts of their keys, `slots` workgroups in all or fewer; launch(parts, blocks, records) of tiles
// of `rows` rows.
template <int HD, int K, int R, class Launch>
int tree_launch(const AttnKv &c, float *out, int64_t ldo, const int *slot, const int *base, const uint64_t *seen, int n_seq, int N,
                int H, int rows, int64_t slots, Launch launch) {
	const int64_t tiles = ((int64_t)N * (H / c.kvh) + rows - 1) / rows, wgs = tiles * n_seq * c.kvh;
	const int most = (tile_steps<K>(c.max_seq, c.prefix_len) + R - 1) / R;
	// (whole rounds of the eight dies: one tree of 448 rows at 8000, four heads, 41 us in 9 parts, 31 in 8. As many parts for
	// all as fit at once: trees of 64 at 4096, four heads, fill the chip at 16, 126 us in two parts; 17 are one part, 136
	// workgroups in 183 us, and 33 a second round, 395)
	const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(most, slots / (8 * tiles) * 8 / ((int64_t)n_seq * c.kvh)));
	if ((wgs * parts + 8 * tiles) > kMaxThreads / 512 || (int64_t)n_seq * N * H * (HD / 4) > kMaxThreads)
		return set_error(HAKO_GPU_EINVAL, "%lld workgroups in one call", (long long)(wgs * parts));
	Records rec{};
	if (parts > 1)
		if (int rc = records((size_t)n_seq * N * H * parts, HD, &rec)) return rc;
	launch(parts, dim3(tree_blocks((int64_t)n_seq * c.kvh * parts, tiles)), rec);
	HK_LAUNCHED("attention");
	// many parts, or rows so few that the other join's would be alone with them (3B heads, us by the other / this: one tree of
	// 4 nodes at 32000 in 64 parts 77 / 21, of 26 at 1025 in 9 12.9 / 12.0, but 8 of 64 at 4000 in 8 50 / 53)
	if (parts > 16 || (parts > 6 && (int64_t)n_seq * N * H <= 1024)) {
		hipLaunchKernelGGL((tree_join_wide_kernel<HD, K, R>), dim3(H, n_seq * N), dim3(64 * kJoin), 0, stream(), c, out, ldo, slot, base, seen, N, parts,
		                   rec.o, rec.ml, rec.e);
		HK_LAUNCHED("attention join");
	} else if (parts > 1) {
		const int64_t blocks = ((int64_t)n_seq * N * H * (HD / 4) + 255) / 256;
		hipLaunchKernelGGL((tree_join_kernel<HD, K, R>), dim3((unsigned)blocks), dim3(256), 0, stream(), c, out, ldo, slot, base, seen, n_seq, N,
		                   H, parts, rec.o, rec.ml, rec.e);
		HK_LAUNCHED("attention join");
	}
	return HAKO_GPU_OK;
}

// Which kernel (one MI355X, us a call by the direct / the tiled one; the texts fill their slots). Lengths are known on the device
// alone, so the work is taken as if slots were full: shorter texts may then take the tiled kernel, at up to 10 us more.
//   rows of a sequence and head   wave-steps a SIMD (32 rows x 32 keys)   8 bits       16 bits
//   7B  8 trees of 64 at 1000  448 rows     14                          33 / 39      36 / 39
//       8 of 32 at 4000        224          28                          56 / 48      61 / 50
//       16 of 64 at 4096       448         112                         168 / 124    189 / 134
//       8 of 16 at 2000        112           8                          25 / 33      27 / 33
//       16 of 12 at 4000        84          24                          54 / 51      59 / 51
//       32 of 16 at 3400       112          54                          82 / 79      94 / 84
//       64 of 16 at 2000       112          64                          98 / 91     120 / 96
//       64 of 8 at 2000         56          32                          56 / 77      68 / 78
//   3B  8 of 64 at 4000        512          32                          58 / 52      63 / 53
// So the tiled one from 24 on for more than 64 rows. Its tiles are of 128 rows where these hold them all and sequences and
// heads do not give every other CU a tile (32 ragged trees of 16 over a prefix in 16 bits 62 us, 72 in tiles of 256, 8
// bits 65 and 74; 64 of 16 at 2000 103 and 96, in 8 bits 89 and 91).
template <int HD, bool Q8>
int tree(const AttnKv &c, float *out, int64_t ldo, const float *q, int64_t ldq, const int *slot, const int *base, const uint64_t *seen,
         int n_seq, int N, int H, float scale) {
	const int G = H / c.kvh, rows = N * G;
	const int64_t steps = (int64_t)(rows + 31) / 32 * n_seq * c.kvh * tile_steps<32>(c.max_seq, c.prefix_len);
	const bool tiled = rows > 64 && steps >= 24 * 4 * (int64_t)cu_count();
	const int kernel = g_attn_prompt ? g_attn_prompt : !tiled ? 1 : rows > 128 || 2 * (int64_t)n_seq * c.kvh > cu_count() ? 2 : 3;
	if (kernel == 2)
		return tree_launch<HD, kKeys, 1>(c, out, ldo, slot, base, seen, n_seq, N, H, 256, cu_count(), [&](int parts, dim3 grid, const Records &rec) {
			hipLaunchKernelGGL((tree_tiled_kernel<HD, Q8, 8>), grid, dim3(512), 0, stream(), c, out, ldo, q, ldq, slot, base, seen, n_seq, N, G,
			                   scale * kLog2e, parts, rec);
		});
	if (kernel == 3)
		return tree_launch<HD, kKeys, 1>(c, out, ldo, slot, base, seen, n_seq, N, H, 128, 2 * cu_count(), [&](int parts, dim3 grid, const Records &rec) {
			hipLaunchKernelGGL((tree_tiled_kernel<HD, Q8, 4>), grid, dim3(256), 0, stream(), c, out, ldo, q, ldq, slot, base, seen, n_seq, N, G,
			                   scale * kLog2e, parts, rec);
		});
	return tree_launch<HD, 32, kWaves>(c, out, ldo, slot, base, seen, n_seq, N, H, 32, 2 * cu_count(), [&](int parts, dim3 grid, const Records &rec) {
		hipLaunchKernelGGL((tree_kernel<HD, Q8>), grid, dim3(64 * kWaves), 0, stream(), c, out, ldo, q, ldq, slot, base, seen, n_seq, N, G,
		                   scale * kLog2e, parts, rec);
	});
}

}  // namespace

int attn_decode(float *out, int64_t ldo, const float *q, int64_t ldq, const hako_gpu_kv *kv, const int *slot,
                const int *len, int len_add, int n_seq, int H, float scale, int prefix_slot, int prefix_len) {
	const AttnKv c = attn_kv(kv, prefix_slot, prefix_len, len_add);
#define HK_DECODE(HD, Q8) decode<HD, Q8, false>(c, out, ldo, q, ldq, slot, len, n_seq, H, scale)
	return HK_KV_SWITCH(kv, HK_DECODE);
#undef HK_DECODE
}

int attn_decode_window(float *out, int64_t ldo, const float *q, int64_t ldq, const hako_gpu_kv *kv, const int *slot,
                       const int *len, int len_add, int n_seq, int H, float scale, int window, int sinks) {
	const AttnKv c = attn_kv_window(kv, len_add, window, sinks);
#define HK_DECODE(HD, Q8) decode<HD, Q8, true>(c, out, ldo, q, ldq, slot, len, n_seq, H, scale)
	return HK_KV_SWITCH(kv, HK_DECODE);
#undef HK_DECODE
}

int attn_decode_reserve(const hako_gpu_kv *kv, int n_seq, int H, int prefix_len, int window, int sinks) {
	const AttnKv c = window ? attn_kv_window(kv, 0, window, sinks) : attn_kv(kv, 0, prefix_len, 0);
	const DecodePlan p = decode_plan(most_keys(c), prefix_len, kv->n_kv_heads, n_seq, H, window > 0);
	Records r;
	return p.nrec ? records((size_t)n_seq * H * p.nrec, kv->head_dim, &r) : HAKO_GPU_OK;
}

void attn_set_prompt(int v) { g_attn_prompt = v >= 1 && v <= 3 ? v : 0; }

}  // namespace hako

using namespace hako;

namespace {

int decode_check(const hako_gpu_kv *kv, const int *slot, const int *len, int n_seq) {
	if (!len && n_seq) return set_error(HAKO_GPU_EINVAL, "null lengths");
	if (!slot && n_seq > kv->n_slots)
		return set_error(HAKO_GPU_EINVAL, "%d sequences without slots in a cache of %d", n_seq, kv->n_slots);
	if (n_seq > 65535) return set_error(HAKO_GPU_EINVAL, "%d sequences in one call (at most 65535)", n_seq);
	return HAKO_GPU_OK;
}

int window_check(int window, int sinks) {
	if (window < 1 || sinks < 0) return set_error(HAKO_GPU_EINVAL, "a window of %d positions after %d sinks", window, sinks);
	return HAKO_GPU_OK;
}

// The prompts of a call, checked but for q, out and the cache; rows of q and out.
int prompt_check(const hako_gpu_kv *kv, const int *slot, const int *start, const int *len, int n_seq) {
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
	return HAKO_GPU_OK;
}

int prompts(const AttnKv &c, const hako_gpu_kv *kv, float *out, int64_t ldo, const float *q, int64_t ldq, const int *slot,
            const int *start, const int *len, int n_seq, int H, float scale) {
	// the sequences with tokens, those that end last (the longest tiles) first
	std::vector<int> order, row;
	try {
		row.resize(n_seq);
		order.reserve(n_seq);
	} catch (const std::bad_alloc &) {
		return set_error(HAKO_GPU_ENOMEM, "host memory for %d sequences", n_seq);
	}
	for (int s = 0, r = 0; s < n_seq; r += len[s++]) {
		row[s] = r;
		if (len[s]) order.push_back(s);
	}
	std::sort(order.begin(), order.end(), [&](int a, int b) {
		const int ea = start[a] + len[a], eb = start[b] + len[b];
		return ea != eb ? ea > eb : a < b;
	});
	for (size_t i = 0; i < order.size();) {
		SeqTab t{};
		for (; i < order.size() && t.n < kSeqs; i++, t.n++) {
			const int s = order[i];
			t.row[t.n] = row[s];
			t.len[t.n] = len[s];
			t.slot[t.n] = slot ? slot[s] : s;
			t.start[t.n] = start[s];
		}
#define HK_PROMPT(HD, Q8) (c.window ? prompt<HD, Q8, true>(c, t, out, ldo, q, ldq, H, scale) : prompt<HD, Q8, false>(c, t, out, ldo, q, ldq, H, scale))
		if (int rc = HK_KV_SWITCH(kv, HK_PROMPT)) return rc;
#undef HK_PROMPT
	}
	return HAKO_GPU_OK;
}

}  // namespace

extern "C" {

int hako_gpu_attn_decode(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                         const int *slot, const int *len, int n_seq, int n_heads, float scale, int prefix_slot,
                         int prefix_len) {
	if (int rc = attn_check(out, out_stride, q, q_stride, kv, n_seq, n_heads, prefix_slot, prefix_len)) return rc;
	if (int rc = decode_check(kv, slot, len, n_seq)) return rc;
	if (int rc = require_device()) return rc;
	if (n_seq == 0) return ok();
	if (int rc = attn_decode(out, out_stride, q, q_stride, kv, slot, len, 0, n_seq, n_heads, scale, prefix_slot, prefix_len))
		return rc;
	return ok();
}

int hako_gpu_attn_decode_window(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                                const int *slot, const int *len, int n_seq, int n_heads, float scale, int window,
                                int sinks) {
	if (int rc = attn_check(out, out_stride, q, q_stride, kv, n_seq, n_heads, 0, 0)) return rc;
	if (int rc = decode_check(kv, slot, len, n_seq)) return rc;
	if (int rc = window_check(window, sinks)) return rc;
	if (int rc = require_device()) return rc;
	if (n_seq == 0) return ok();
	if (int rc = attn_decode_window(out, out_stride, q, q_stride, kv, slot, len, 0, n_seq, n_heads, scale, window, sinks)) return rc;
	return ok();
}

int hako_gpu_attn_prompt(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                         const int *slot, const int *start, const int *len, int n_seq, int n_heads, float scale,
                         int prefix_slot, int prefix_len) {
	if (int rc = attn_check(out, out_stride, q, q_stride, kv, n_seq, n_heads, prefix_slot, prefix_len)) return rc;
	if (int rc = prompt_check(kv, slot, start, len, n_seq)) return rc;
	if (int rc = require_device()) return rc;
	if (int rc = prompts(attn_kv(kv, prefix_slot, prefix_len, 0), kv, out, out_stride, q, q_stride, slot, start, len, n_seq, n_heads, scale))
		return rc;
	return ok();
}

int hako_gpu_attn_prompt_window(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                                const int *slot, const int *start, const int *len, int n_seq, int n_heads, float scale,
                                int window, int sinks) {
	if (int rc = attn_check(out, out_stride, q, q_stride, kv, n_seq, n_heads, 0, 0)) return rc;
	if (int rc = prompt_check(kv, slot, start, len, n_seq)) return rc;
	if (int rc = window_check(window, sinks)) return rc;
	if (int rc = require_device()) return rc;
	if (int rc = prompts(attn_kv_window(kv, 0, window, sinks), kv, out, out_stride, q, q_stride, slot, start, len, n_seq, n_heads, scale))
		return rc;
	return ok();
}

int hako_gpu_attn_tree(float *out, int64_t out_stride, const float *q, int64_t q_stride, const hako_gpu_kv *kv,
                       const int *slot, const int *base, const uint64_t *seen, int n_seq, int n_tree, int n_heads,
                       float scale, int prefix_slot, int prefix_len) {
	if (int rc = attn_check(out, out_stride, q, q_stride, kv, n_seq, n_heads, prefix_slot, prefix_len)) return rc;
	if (int rc = tree_check(n_seq, n_tree)) return rc;
	if (n_seq && (!base || !seen)) return set_error(HAKO_GPU_EINVAL, "null bases or masks");
	if ((uintptr_t)seen & 7) return set_error(HAKO_GPU_EINVAL, "masks are not 8-byte aligned");
	if (!slot && n_seq > kv->n_slots)
		return set_error(HAKO_GPU_EINVAL, "%d sequences without slots in a cache of %d", n_seq, kv->n_slots);
	if (int rc = require_device()) return rc;
	if (n_seq == 0) return ok();
	const AttnKv c = attn_kv(kv, prefix_slot, prefix_len, 0);
#define HK_TREE(HD, Q8) tree<HD, Q8>(c, out, out_stride, q, q_stride, slot, base, seen, n_seq, n_tree, n_heads, scale)
	if (int rc = HK_KV_SWITCH(kv, HK_TREE)) return rc;
#undef HK_TREE
	return ok();
}

}  // extern "C"
