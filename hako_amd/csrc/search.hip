// search.hip — beams and drafted trees (include/hako_search.h): the choice of
// continuations from a step's logits, a tree's plan and its accepted path, and
// the cache rows that move after either.
#include "kv.h"

#include "../../include/hako_search.h"

namespace hako {
namespace {

constexpr int kWsSearch = 8;   // library workspace slot of the selection's parts
constexpr int kLayers = 32;    // caches of one launch (by value in the kernel arguments)
constexpr float kInf = __builtin_inff();

// What a wave wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync() {
	__builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
	__builtin_amdgcn_wave_barrier();
	__builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ int lanes_below(uint64_t m) {
	return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// ── the n best of a stream of values, by one wave ──
//
// Values come in tiles of 64 E, position (i 64 + lane) 4 + c of a tile in
// register 4 i + c; equal ones rank by position, or by ids that rise with it
// (register e's is id(e)). Of a tile only what may still
// be among the n best is kept: values above the n-th best known so far, and
// where more than n lanes have such values, above the n-th largest of the
// lanes' own maxima, or what tells it from the next (found bit by bit, a
// ballot each), which at most n lanes exceed. So no tile adds more than
// n (E + 1), whatever the values are, and an ordinary one about n at first and
// hardly any later. What is kept waits in LDS until there are more than 64, and
// is then ranked: a lane a value, each against all, as 64-bit keys of value and
// position.
template <int E>
struct Best {
	struct Lds {
		alignas(16) uint64_t key[64 + HAKO_MAX_PICK * (E + 1) + 4], list[HAKO_MAX_PICK];
	};
	int n, count;   // wanted, waiting
	float least;    // a later value has to be larger

	// (zeros of both signs are equal)
	static __device__ __forceinline__ uint64_t key_of(float v, int id) {
		const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
		return (uint64_t)(b >> 31 ? ~b : b | 0x80000000u) << 32 | (uint32_t)~id;
	}
	static __device__ __forceinline__ float value(uint64_t key) {
		const uint32_t k = (uint32_t)(key >> 32);
		return __builtin_bit_cast(float, k >> 31 ? k & 0x7FFFFFFFu : ~k);
	}
	static __device__ __forceinline__ int id_of(uint64_t key) { return (int)~(uint32_t)key; }

	__device__ __forceinline__ void start(int want) {
		n = want;
		count = 0;
		least = -kInf;
	}

	// A place of a tile from pos0.
	static __device__ __forceinline__ int pos(int e, int pos0, int lane) { return pos0 + ((e >> 2) * 64 + lane) * 4 + (e & 3); }

	// mx: the lane's largest value
	template <class Id>
	__device__ __forceinline__ void tile(const float (&x)[E], float mx, const Id &id, Lds &s, int lane) {
		const uint64_t hits = __ballot(mx > least);
		if (!hits) return;
		float t = least;
		int ties = 0;   // values equal to t that may come in, the first ones
		if (__popcll(hits) > n) {
			const uint32_t key = (uint32_t)(key_of(mx, 0) >> 32);
			uint32_t k = 0;
			for (int bit = 31; bit >= 0; bit--) {
				const uint32_t up = k | 1u << bit;
				const int above = __popcll(__ballot(key >= up));
				k = above >= n ? up : k;
				if (above == n) break;
			}
			t = value((uint64_t)k << 32);
			ties = n;
		}
		int c = count;
#pragma unroll
		for (int e = 0; e < E; e++) {
			const uint64_t m = __ballot(x[e] > t);
			if (!m) continue;
			if (x[e] > t) s.key[c + lanes_below(m)] = key_of(x[e], id(e));
			c += __popcll(m);
		}
		if (ties) {
#pragma unroll
			for (int g = 0; g < E; g += 4) {   // in the order of the positions
				uint64_t m[4];
				int before = 0, all = 0;
#pragma unroll
				for (int e = 0; e < 4; e++) {
					m[e] = __ballot(x[g + e] == t);
					before += lanes_below(m[e]);
					all += __popcll(m[e]);
				}
				if (!all || ties <= 0) continue;
#pragma unroll
				for (int e = 0; e < 4; e++)
					if (x[g + e] == t) {
						if (before < ties) s.key[c + before] = key_of(t, id(g + e));
						before++;
					}
				c += min(all, ties);
				ties -= all;
			}
		}
		count = c;
		if (c > 64 || (c >= n && least == -kInf)) settle(s, lane);
	}

	// The n best of what waits, in order, in list (and waiting again).
	__device__ __forceinline__ void settle(Lds &s, int lane) {
		if (lane < 4) s.key[count + lane] = 0;
		wave_sync();
		for (int j = lane; j < count; j += 64) {
			const uint64_t mine = s.key[j];
			int rank = 0;
			for (int k = 0; k < count; k += 4) {
				const ulonglong2 a = *(const ulonglong2 *)(s.key + k), b = *(const ulonglong2 *)(s.key + k + 2);
				rank += (a.x > mine) + (a.y > mine) + (b.x > mine) + (b.y > mine);
			}
			if (rank < n) s.list[rank] = mine;
		}
		wave_sync();
		count = min(count, n);
		if (lane < count) s.key[lane] = s.list[lane];
		if (count == n) least = value(s.list[n - 1]);
	}
};

// ── beam selection ──
//
// value(b, t) = score_b + (x_bt - log sum_j exp x_bj). Within a beam the order
// is that of the logits, so a pass over them keeps the n largest and the sum,
// and values are formed for n_beams n_pick candidates alone. Two launches:
// waves over parts of the rows (whole tiles, as many as fill the chip with 16
// waves a CU), then a workgroup a request.
// exp sums are taken against the part's maximum, in fp32 with the argument's
// rounding put right, four at a time into 64 bits, and meet in 64 bits.
//
// Bound: no one thing. 32 requests of 8 beams over 152064 tokens (140 MB: the
// tenth of the beams that have ended are not read) take 33.6 us, 4.2 TB/s (a copy
// of 1 GiB 5.0), and the choice 6.7. Where calls follow each other 66 MB come
// from HBM, the rest from the memory-side cache; of 48 wave cycles 23 are waits
// and 11 vector instructions. On the way, in all: every tile's candidates
// ranked as they came 91 us; 64 at a time as 64-bit keys, 16 waves a CU in the
// place of 8, 42. The bound found two bits at a time was slower, as was ranking
// the lanes' maxima in LDS (36.5 us against 33.7).
constexpr int kPickE = 16;                 // values of a lane's tile
constexpr int kPickTile = 64 * kPickE;
constexpr int kPickWaves = 4;
constexpr int kPickFill = 16;              // waves a CU

// Per row and part: the largest value, the sum of exp(x - it), n_pick values
// and their tokens, best first, -inf where there are fewer.
struct Parts {
	double *sum;
	float *top, *v;
	int *i;
};

// exp(d), d <= 0: 2^t (1 + s), s = d - t log(2) what t's rounding left out.
__device__ __forceinline__ float exp_(float d) {
	d = __builtin_fmaxf(d, -104.0f);   // (0 from there on, -inf among them)
	const float t = d * 1.44269504f;
	const float e = __builtin_amdgcn_exp2f(t);
	return __builtin_fmaf(e, __builtin_fmaf(t, -0.693147181f, d), e);
}

// The larger of two, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__global__ __launch_bounds__(64 * kPickWaves) void beam_part_kernel(const float *__restrict__ logits, int64_t ld, int vocab,
                                                                    const int *__restrict__ done, int parts, int span,
                                                                    int n_pick, Parts out) {
	__shared__ typename Best<kPickE>::Lds lds[kPickWaves];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int part = blockIdx.x * kPickWaves + wave;
	const int64_t row = blockIdx.y;
	if (part >= parts || (done && done[row])) return;
	const int from = part * span, n = min(vocab - from, span);
	const __amdgpu_buffer_rsrc_t r = stream_rsrc(uniform_ptr(logits + row * ld + from), (uint32_t)n * 4u);
	Best<kPickE> best;
	best.start(n_pick);
	float top = -kInf;
	double sum = 0.0;
	float x[kPickE], y[kPickE];
	auto load = [&](float(&z)[kPickE], int t) {
#pragma unroll
		for (int g = 0; g < kPickE / 4; g++) {
			const uint4 w = ld_b128(r, 4u * (uint32_t)(t + (g * 64 + lane) * 4));
			z[4 * g] = __builtin_bit_cast(float, w.x);
			z[4 * g + 1] = __builtin_bit_cast(float, w.y);
			z[4 * g + 2] = __builtin_bit_cast(float, w.z);
			z[4 * g + 3] = __builtin_bit_cast(float, w.w);
		}
	};
	auto use = [&](float(&z)[kPickE], int t) {
		if (t + kPickTile > n) {
#pragma unroll
			for (int e = 0; e < kPickE; e++) z[e] = best.pos(e, t, lane) < n ? z[e] : -kInf;
		}
		float mx = z[0];
#pragma unroll
		for (int e = 1; e < kPickE; e++) mx = max_nan(mx, z[e]);
		if (__any(mx != mx)) {   // the row has no continuations, whatever else it holds
			sum = __builtin_nan("");
			return;
		}
		const float m = wave_max(mx);
		if (m > top) {
			sum *= exp((double)top - (double)m);
			top = m;
		}
		if (top > -kInf) {
#pragma unroll
			for (int e = 0; e < kPickE; e += 4)
				sum += (double)((exp_(z[e] - top) + exp_(z[e + 1] - top)) + (exp_(z[e + 2] - top) + exp_(z[e + 3] - top)));
		}
		best.tile(z, mx, [&](int e) { return best.pos(e, from + t, lane); }, lds[wave], lane);
	};
	load(x, 0);
	for (int t = 0; t < n; t += 2 * kPickTile) {
		if (t + kPickTile < n) load(y, t + kPickTile);
		use(x, t);
		if (t + kPickTile >= n) break;
		if (t + 2 * kPickTile < n) load(x, t + 2 * kPickTile);
		use(y, t + kPickTile);
	}
	best.settle(lds[wave], lane);
#pragma unroll
	for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k);
	const int64_t rec = row * parts + part;
	if (lane == 0) {
		out.top[rec] = top;
		out.sum[rec] = sum;
	}
	if (lane < n_pick) {
		const uint64_t key = lane < best.count ? lds[wave].list[lane] : 0;
		out.v[rec * n_pick + lane] = lane < best.count ? best.value(key) : -kInf;
		out.i[rec * n_pick + lane] = best.id_of(key);
	}
}

// The join, a wave a beam: its sum and its n_pick best; then the request's best
// of those. Bound by latency: all that it reads is asked for at once (one
// request of 4 beams in 149 parts 6.1 us, 6.9 when sums of parts past the 64th
// and the chosen ones' tokens were asked for later), and its code is short
// where it may be (tiles of 512 values 7.0 us for 32 requests of 8 beams, of
// 256 6.7).
constexpr int kJoinE = 4;
constexpr int kJoinR = 3;   // rounds of parts whose sums are asked for at once

__global__ __launch_bounds__(64 * HAKO_MAX_BEAMS) void beam_join_kernel(const float *__restrict__ score, const int *__restrict__ done,
                                                                        int eos, int n_beams, int n_pick, int parts, int arrange,
                                                                        Parts in, int *__restrict__ parent, int *__restrict__ token,
                                                                        float *__restrict__ score_out, int *__restrict__ done_out) {
	__shared__ typename Best<kJoinE>::Lds lds[HAKO_MAX_BEAMS];
	__shared__ double val[HAKO_MAX_BEAMS * HAKO_MAX_PICK];
	__shared__ int tok[HAKO_MAX_BEAMS * HAKO_MAX_PICK], rank[HAKO_MAX_BEAMS * HAKO_MAX_PICK], pick[HAKO_MAX_PICK], over[HAKO_MAX_BEAMS];
	const int lane = threadIdx.x & 63, b = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int64_t req = blockIdx.x, row = req * n_beams + b;
	const double old = (double)score[row];
	const int ended = done ? done[row] : 0;
	// the parts' lists in the order of their tokens; in a list equal values are in that order too (values and tokens come
	// together, so that nothing is looked up for what was chosen)
	const int64_t rec = row * parts;
	const int n_list = parts * n_pick;
	const __amdgpu_buffer_rsrc_t r = stream_rsrc(uniform_ptr(in.v + rec * n_pick), (uint32_t)n_list * 4u);
	const __amdgpu_buffer_rsrc_t ri = stream_rsrc(uniform_ptr(in.i + rec * n_pick), (uint32_t)n_list * 4u);
	float x[kJoinE];
	int id[kJoinE];
	auto load = [&](int t) {
#pragma unroll
		for (int g = 0; g < kJoinE / 4; g++) {
			const uint32_t at = 4u * (uint32_t)(t + (g * 64 + lane) * 4);
			const uint4 w = ld_b128(r, at), i = ld_b128(ri, at);
			const float z[4] = {__builtin_bit_cast(float, w.x), __builtin_bit_cast(float, w.y), __builtin_bit_cast(float, w.z), __builtin_bit_cast(float, w.w)};
			const uint32_t j[4] = {i.x, i.y, i.z, i.w};
#pragma unroll
			for (int e = 0; e < 4; e++) {
				x[4 * g + e] = z[e];
				id[4 * g + e] = (int)j[e];
			}
		}
	};
	load(0);
	// (an ended beam's are whatever was there)
	float tops[kJoinR];
	double sums[kJoinR];
#pragma unroll
	for (int k = 0; k < kJoinR; k++) {
		const int p = k * 64 + lane;
		tops[k] = p < parts ? in.top[rec + p] : -kInf;
		sums[k] = p < parts ? in.sum[rec + p] : 0.0;
	}
	if (threadIdx.x < HAKO_MAX_PICK) pick[threadIdx.x] = -1;
	if (lane == 0) over[b] = ended;
	if (ended) {
		if (lane < n_pick) {
			val[b * n_pick + lane] = lane == 0 ? old : -(double)kInf;
			tok[b * n_pick + lane] = eos;
		}
	} else {
		float top = tops[0];
#pragma unroll
		for (int k = 1; k < kJoinR; k++) top = __builtin_fmaxf(top, tops[k]);
		for (int p = kJoinR * 64 + lane; p < parts; p += 64) top = __builtin_fmaxf(top, in.top[rec + p]);
		top = wave_max(top);
		double sum = 0.0;
		auto add = [&](float t, double w) { sum += t == -kInf ? w : w * (double)exp_(t - top); };
#pragma unroll
		for (int k = 0; k < kJoinR; k++) add(tops[k], sums[k]);
		for (int p = kJoinR * 64 + lane; p < parts; p += 64) add(in.top[rec + p], in.sum[rec + p]);
#pragma unroll
		for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k);
		const double lse = (double)top + log(sum);
		Best<kJoinE> best;
		best.start(n_pick);
		for (int t = 0; t < n_list; t += 64 * kJoinE) {
			float mx = -kInf;
#pragma unroll
			for (int e = 0; e < kJoinE; e++) {
				x[e] = best.pos(e, t, lane) < n_list ? x[e] : -kInf;
				mx = __builtin_fmaxf(mx, x[e]);
			}
			best.tile(x, mx, [&](int e) { return id[e]; }, lds[b], lane);
			if (t + 64 * kJoinE < n_list) load(t + 64 * kJoinE);
		}
		best.settle(lds[b], lane);
		if (lane < n_pick) {
			const bool on = lane < best.count;
			const uint64_t key = on ? lds[b].list[lane] : 0;
			val[b * n_pick + lane] = on ? old + ((double)best.value(key) - lse) : -(double)kInf;
			tok[b * n_pick + lane] = on ? best.id_of(key) : -1;
		}
	}
	const int n = n_beams * n_pick;
	if (lane < n_pick) rank[b * n_pick + lane] = 0;
	__syncthreads();
	// How many of this wave's list go before each value: the lists fall (so that a place in one stands for logits and
	// tokens), and equal values go by list.
	for (int f = lane; f < n; f += 64) {
		const double v = val[f];
		const int own = f - b * n_pick;
		int before = 0;
#pragma unroll
		for (int step = HAKO_MAX_PICK; step; step >>= 1) {
			const double x = val[b * n_pick + min(before + step, n_pick) - 1];
			before += before + step <= n_pick && (x > v || (x == v && own >= 0)) ? step : 0;
		}
		atomicAdd(&rank[f], own >= 0 && own < n_pick ? own : before);
	}
	__syncthreads();
	for (int f = threadIdx.x; f < n; f += blockDim.x)
		if (val[f] > -(double)kInf && rank[f] < n_pick) pick[rank[f]] = f;
	__syncthreads();
	if (threadIdx.x >= 64) return;
	const int f = lane < n_pick ? pick[lane] : -1, from = f < 0 ? -1 : f / n_pick;
	int place = lane;
	if (arrange) {
		uint32_t taken = 0;
		bool first = false;
		for (int k = 0; k < n_beams; k++) {
			const uint64_t m = __ballot(from == k);
			if (m) taken |= 1u << k;
			if (from == k) first = __ffsll((unsigned long long)m) - 1 == lane;
		}
		const uint64_t rest = __ballot(lane < n_pick && !first);
		uint32_t left = ~taken;
		for (int k = lanes_below(rest); k > 0; k--) left &= left - 1;
		place = first ? from : __builtin_ctz(left | 1u << 31);
	}
	if (lane >= n_pick) return;
	const int64_t o = req * n_pick + place;
	const int t = f < 0 ? -1 : tok[f];
	parent[o] = from;
	token[o] = t;
	score_out[o] = f < 0 ? -kInf : (float)val[f];
	if (done_out) done_out[o] = f >= 0 && (t == eos || over[from]);
}

// ── cache rows that move ──

// The caches of a launch: codes, then scales, of one shape.
struct Layers {
	uint8_t *k[kLayers], *v[kLayers];
	float *ks[kLayers], *vs[kLayers];
};
struct Shape {
	int n_slots, max_seq, kvh, row;   // row: bytes of a row's codes
};

// A workgroup takes units of 16 bytes (and scales) of one head's rows in all
// of a request's slots at once: every load comes before the first store, so any
// map of places is good, and a source that several places take is read once.
//
// Bound: HBM. 4 requests of 8 beams, 12 layers of 4 heads in 16 bits, half of
// the places moved: 96 MB from memory and 192 MB to it in 68 us, 4.2 TB/s (a
// copy of 1 GiB 5.0), waits three quarters of the waves' cycles. Units as vectors of the compiler (131
// us as structs, whose copies became single words), stores past the caches (82
// without).
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
template <int B>
__global__ __launch_bounds__(256) void reorder_kernel(Layers layers, Shape c, const int *__restrict__ slot,
                                                      const int *__restrict__ parent, int n_beams,
                                                      const int *__restrict__ since, const int *__restrict__ len) {
	const int req = blockIdx.y, z = blockIdx.x, is_v = z & 1, head = (z >> 1) % c.kvh, layer = (z >> 1) / c.kvh;
	const int from = max(since ? since[req] : 0, 0), to = min(len[req], c.max_seq);
	if (from >= to) return;
	// the places that change: their bases, and their sources'
	int64_t dst[B], src[B];   // in rows; -1: stays
	bool any = false;
#pragma unroll
	for (int b = 0; b < B; b++) {
		dst[b] = src[b] = -1;
		if (b >= n_beams) continue;
		const int at = req * n_beams, p = parent[at + b];
		if (p < 0 || p >= n_beams || p == b) continue;
		const int d = slot ? slot[at + b] : at + b, s = slot ? slot[at + p] : at + p;
		if (d < 0 || d >= c.n_slots || s < 0 || s >= c.n_slots) continue;
		dst[b] = ((int64_t)d * c.kvh + head) * c.max_seq;
		src[b] = ((int64_t)s * c.kvh + head) * c.max_seq;
		any = true;
	}
	if (!any) return;
	uint8_t *codes = is_v ? layers.v[layer] : layers.k[layer];
	float *scales = is_v ? layers.vs[layer] : layers.ks[layer];
	const int64_t units = (int64_t)(to - from) * (c.row / 16), first = (int64_t)from * (c.row / 16);
	for (int64_t u = (int64_t)blockIdx.z * 256 + threadIdx.x; u < units; u += (int64_t)gridDim.z * 256) {
		u4 x[B];
#pragma unroll
		for (int b = 0; b < B; b++)
			if (src[b] >= 0) x[b] = *(const u4 *)(codes + src[b] * c.row + 16 * (first + u));
#pragma unroll
		for (int b = 0; b < B; b++)
			if (src[b] >= 0) __builtin_nontemporal_store(x[b], (u4 *)(codes + dst[b] * c.row + 16 * (first + u)));
	}
	for (int64_t u = (int64_t)blockIdx.z * 256 + threadIdx.x; u < to - from; u += (int64_t)gridDim.z * 256) {
		float x[B];
#pragma unroll
		for (int b = 0; b < B; b++)
			if (src[b] >= 0) x[b] = scales[src[b] + from + u];
#pragma unroll
		for (int b = 0; b < B; b++)
			if (src[b] >= 0) scales[dst[b] + from + u] = x[b];
	}
}

// A wave takes a path's rows of one head, keys or values: all of its loads,
// then its stores, so that a row may be another one's place. Bound by latency:
// a path is at most 16 KB a head, 28 layers of 32 paths of 1..9 rows (10.9 MB)
// 7.4 us, 12 layers of one path 4.3: the path, its rows, their stores, one
// after the other.
constexpr int kKeepWaves = 4;
__global__ __launch_bounds__(64 * kKeepWaves) void keep_kernel(Layers layers, Shape c, int n_layers, const int *__restrict__ slot,
                                                               const int *__restrict__ base, const int *__restrict__ path,
                                                               const int *__restrict__ n_path, int n_tree) {
	const int sq = blockIdx.y, lane = threadIdx.x & 63;
	const int z = __builtin_amdgcn_readfirstlane(blockIdx.x * kKeepWaves + (threadIdx.x >> 6));
	const int is_v = z & 1, head = (z >> 1) % c.kvh, layer = (z >> 1) / c.kvh;
	if (layer >= n_layers) return;
	const int sl = slot ? slot[sq] : sq, b = base[sq], n = min(n_path[sq], n_tree);
	if (sl < 0 || sl >= c.n_slots || b < 0) return;
	// lane d: where row d comes from, -1: it stays
	int from = lane < n ? path[(int64_t)sq * n_tree + lane] : -1;
	if (from < 0 || from >= n_tree || from == lane || b > c.max_seq - 1 - max(from, lane)) from = -1;
	const uint64_t moves = __ballot(from >= 0);
	if (!moves) return;
	const int64_t r = ((int64_t)sl * c.kvh + head) * c.max_seq + b;
	uint8_t *codes = (is_v ? layers.v[layer] : layers.k[layer]) + r * c.row;
	float *scales = (is_v ? layers.vs[layer] : layers.ks[layer]) + r;
	const int units = c.row / 16, lg = __builtin_ctz(units), rows = 64 - __builtin_clzll(moves);   // (rows past the last that moves stay)
	float y = 0.0f;
	if (from >= 0) y = scales[from];
	uint4 x[16];
#pragma unroll
	for (int i = 0; i < 16; i++) {
		const int u = i * 64 + lane, d = u >> lg, f = __shfl(from, d & 63);
		x[i] = make_uint4(0, 0, 0, 0);
		if (i * 64 < rows * units && d < rows && f >= 0) x[i] = *(const uint4 *)(codes + (int64_t)f * c.row + 16 * (u & (units - 1)));
	}
	// every load's data is here before the first store
	asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
	if (from >= 0) scales[lane] = y;
#pragma unroll
	for (int i = 0; i < 16; i++) {
		const int u = i * 64 + lane, d = u >> lg, f = __shfl(from, d & 63);
		if (i * 64 < rows * units && d < rows && f >= 0) *(uint4 *)(codes + (int64_t)d * c.row + 16 * (u & (units - 1))) = x[i];
	}
}

// ── drafted trees: a wave a tree, a lane a node ──
//
// A plan by pointer doubling, six rounds for 64 nodes, a path by a ballot a
// step; 1.7 and 2.0 us for one tree, which is a launch.

constexpr int kTreeWaves = 4;

__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int lane) {
	return (uint64_t)(uint32_t)__shfl((int)(uint32_t)v, lane) | ((uint64_t)(uint32_t)__shfl((int)(v >> 32), lane) << 32);
}

// Nodes that are there, as a mask: those before the first whose parent is none.
__device__ __forceinline__ uint64_t tree_nodes(int parent, int lane, int n_tree) {
	const uint64_t bad = __ballot(lane >= n_tree || parent < -1 || parent >= lane);
	return bad ? (1ull << (__ffsll((unsigned long long)bad) - 1)) - 1 : ~0ull;
}

__global__ __launch_bounds__(64 * kTreeWaves) void tree_plan_kernel(const int *__restrict__ slot, const int *__restrict__ base,
                                                                    const int *__restrict__ parent, int n_seq, int n_tree,
                                                                    uint64_t *__restrict__ seen, int *__restrict__ node_slot,
                                                                    int *__restrict__ row, int *__restrict__ turn) {
	const int sq = blockIdx.x * kTreeWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
	if (sq >= n_seq) return;
	const int64_t at = (int64_t)sq * n_tree + lane;
	const int b = base[sq], p = lane < n_tree ? parent[at] : -2;
	const uint64_t nodes = tree_nodes(p, lane, n_tree);
	const bool on = nodes >> lane & 1 && b >= 0;
	// a node's mask and the node that its mask leads up to, each round twice as far
	uint64_t m = 1ull << lane;
	int up = on ? p : -1;
#pragma unroll
	for (int k = 0; k < 6; k++) {
		const uint64_t more = shfl_u64(m, up & 63);
		const int next = __shfl(up, up & 63);
		m |= up >= 0 ? more : 0;
		up = up >= 0 ? next : -1;
	}
	if (lane >= n_tree) return;
	if (seen) seen[at] = on ? m : 0;
	if (node_slot) node_slot[at] = slot ? slot[sq] : sq;
	// (a place past what an int holds is outside every cache: none)
	auto after = [&](int k) { return on ? max((int)((uint32_t)b + (uint32_t)k), -1) : -1; };
	if (row) row[at] = after(lane);
	if (turn) turn[at] = after(__popcll(m) - 1);
}

__global__ __launch_bounds__(64 * kTreeWaves) void tree_accept_kernel(const int *__restrict__ parent, const int *__restrict__ token,
                                                                      const int *__restrict__ pick, const int *__restrict__ base,
                                                                      int n_seq, int n_tree, int *__restrict__ path,
                                                                      int *__restrict__ n_path, int *__restrict__ next,
                                                                      int *__restrict__ new_base) {
	const int sq = blockIdx.x * kTreeWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
	if (sq >= n_seq) return;
	const int64_t at = (int64_t)sq * n_tree + lane;
	const bool in = lane < n_tree;
	const int p = in ? parent[at] : -2, t = in ? token[at] : 0, mine = in ? pick[at] : 0;
	const int b = base ? base[sq] : 0;
	const uint64_t nodes = b < 0 ? 0 : tree_nodes(p, lane, n_tree);
	int here = nodes & 1 ? 0 : -1, n = 0, last = -1, step = -1;   // step: this lane's place of the path
	while (here >= 0) {
		if (lane == n) step = here;
		n++;
		last = __shfl(mine, here);
		const uint64_t child = __ballot(p == here && t == last) & nodes;
		here = child ? __ffsll((unsigned long long)child) - 1 : -1;
	}
	if (in) path[at] = step;
	if (lane == 0) {
		n_path[sq] = n;
		next[sq] = last;
		if (new_base) new_base[sq] = b + n;
	}
}

int caches_check(const hako_gpu_kv *kv, int n_kv) {
	if (n_kv < 1 || !kv) return set_error(HAKO_GPU_EINVAL, "%d caches", n_kv);
	for (int i = 0; i < n_kv; i++) {
		if (int rc = kv_check(&kv[i])) return rc;
		if (kv[i].type != kv->type || kv[i].n_slots != kv->n_slots || kv[i].max_seq != kv->max_seq ||
		    kv[i].n_kv_heads != kv->n_kv_heads || kv[i].head_dim != kv->head_dim)
			return set_error(HAKO_GPU_EINVAL, "cache %d is of another shape than the first", i);
	}
	return HAKO_GPU_OK;
}

// launch(layers, n) for up to kLayers caches at a time
template <class Launch>
int each_layers(const hako_gpu_kv *kv, int n_kv, Launch launch) {
	for (int i = 0; i < n_kv; i += kLayers) {
		Layers l{};
		const int n = n_kv - i < kLayers ? n_kv - i : kLayers;
		for (int j = 0; j < n; j++) {
			l.k[j] = (uint8_t *)kv[i + j].k;
			l.v[j] = (uint8_t *)kv[i + j].v;
			l.ks[j] = kv[i + j].k_scale;
			l.vs[j] = kv[i + j].v_scale;
		}
		launch(l, n);
		HK_LAUNCHED("cache rows");
	}
	return HAKO_GPU_OK;
}

Shape shape_of(const hako_gpu_kv *kv) { return {kv->n_slots, kv->max_seq, kv->n_kv_heads, kv->head_dim * kv_elt(kv->type)}; }

// How the rows of a selection are shared out, parts of whole tiles until the waves fill the chip, and the room for them.
int beam_parts(int rows, int vocab, int n_pick, int *span, int *parts, Parts *out) {
	const int tiles = (vocab + kPickTile - 1) / kPickTile, want = (kPickFill * cu_count() + rows - 1) / rows;
	*span = (tiles + want - 1) / want * kPickTile;
	*parts = (vocab + *span - 1) / *span;
	const size_t recs = (size_t)rows * *parts;
	void *p = nullptr;
	if (int rc = workspace(kWsSearch, recs * (12 + 8 * (size_t)n_pick), &p)) return rc;
	out->sum = (double *)p;
	out->top = (float *)(out->sum + recs);
	out->v = out->top + recs;
	out->i = (int *)(out->v + recs * n_pick);
	return HAKO_GPU_OK;
}

// Workgroups of a launch over the heads of its caches, each with n sequences' rows, some to spare.
int heads_check(int n_kv, const Shape &c, int n) {
	const int64_t heads = (int64_t)(n_kv < kLayers ? n_kv : kLayers) * c.kvh * 2 * n;
	if (heads > kMaxThreads / 512) return set_error(HAKO_GPU_EINVAL, "%lld heads of %d sequences in one call", (long long)heads, n);
	return HAKO_GPU_OK;
}

}  // namespace

int beam_reserve(int rows, int vocab, int n_pick) {
	int span, parts;
	Parts out;
	return beam_parts(rows, vocab, n_pick, &span, &parts, &out);
}

int tree_check(int n_seq, int n_tree) {
	if (n_seq < 0 || n_seq > 0x7FFFFFFF / HAKO_MAX_TREE || n_tree < 1 || n_tree > HAKO_MAX_TREE)
		return set_error(HAKO_GPU_EINVAL, "%d trees of %d nodes (1 to %d)", n_seq, n_tree, HAKO_MAX_TREE);
	return HAKO_GPU_OK;
}

}  // namespace hako

using namespace hako;

extern "C" {

int hako_gpu_beam_select(const float *logits, int64_t ld, int vocab, const float *score, const int *done, int eos,
                         int n_req, int n_beams, int n_pick, int arrange, int *parent, int *token, float *score_out,
                         int *done_out) {
	if (n_req < 0 || n_beams < 1 || n_beams > HAKO_MAX_BEAMS || (int64_t)n_req * n_beams > 65535)
		return set_error(HAKO_GPU_EINVAL, "%d requests of %d beams (1 to %d, at most 65535 in all)", n_req, n_beams, HAKO_MAX_BEAMS);
	if (vocab < 1 || vocab > 1 << 24 || ld < vocab)
		return set_error(HAKO_GPU_EINVAL, "a vocabulary of %d (at most %d) in rows of %lld", vocab, 1 << 24, (long long)ld);
	if (n_pick < 1 || n_pick > HAKO_MAX_PICK || (arrange && n_pick != n_beams))
		return set_error(HAKO_GPU_EINVAL, "%d continuations of %d beams%s (1 to %d)", n_pick, n_beams, arrange ? ", arranged" : "",
		                 HAKO_MAX_PICK);
	if (!logits || !score || !parent || !token || !score_out) return set_error(HAKO_GPU_EINVAL, "null argument");
	if (int rc = require_device()) return rc;
	if (n_req == 0) return ok();
	const int rows = n_req * n_beams;
	int span, parts;
	Parts out;
	if (int rc = beam_parts(rows, vocab, n_pick, &span, &parts, &out)) return rc;
	hipLaunchKernelGGL(beam_part_kernel, dim3((parts + kPickWaves - 1) / kPickWaves, rows), dim3(64 * kPickWaves), 0, stream(), logits, ld,
	                   vocab, done, parts, span, n_pick, out);
	HK_LAUNCHED("beam parts");
	hipLaunchKernelGGL(beam_join_kernel, dim3(n_req), dim3(64 * n_beams), 0, stream(), score, done, eos, n_beams, n_pick, parts, arrange,
	                   out, parent, token, score_out, done_out);
	HK_LAUNCHED("beam choice");
	return ok();
}

int hako_gpu_kv_reorder(const hako_gpu_kv *kv, int n_kv, const int *slot, const int *parent, int n_req, int n_beams,
                        const int *since, const int *len) {
	if (int rc = caches_check(kv, n_kv)) return rc;
	if (n_req < 0 || n_beams < 1 || n_beams > HAKO_MAX_BEAMS || n_req > 65535)
		return set_error(HAKO_GPU_EINVAL, "%d requests (at most 65535) of %d beams (1 to %d)", n_req, n_beams, HAKO_MAX_BEAMS);
	if (!slot && (int64_t)n_req * n_beams > kv->n_slots)
		return set_error(HAKO_GPU_EINVAL, "%d requests of %d beams without slots in a cache of %d", n_req, n_beams, kv->n_slots);
	if (n_req && (!parent || !len)) return set_error(HAKO_GPU_EINVAL, "null parents or lengths");
	if (int rc = require_device()) return rc;
	if (n_req == 0 || n_beams == 1) return ok();
	const Shape c = shape_of(kv);
	if (int rc = heads_check(n_kv, c, n_req)) return rc;
	if (int rc = each_layers(kv, n_kv, [&](const Layers &l, int n) {
		    const int64_t heads = (int64_t)n * c.kvh * 2;
		    const int64_t most = ((int64_t)c.max_seq * (c.row / 16) + 255) / 256, fill = 16 * cu_count() / (heads * n_req) + 1;
		    const dim3 grid((unsigned)heads, n_req, (unsigned)(fill < most ? fill : most));
		    if (n_beams <= 4)
			    hipLaunchKernelGGL(reorder_kernel<4>, grid, dim3(256), 0, stream(), l, c, slot, parent, n_beams, since, len);
		    else if (n_beams <= 8)
			    hipLaunchKernelGGL(reorder_kernel<8>, grid, dim3(256), 0, stream(), l, c, slot, parent, n_beams, since, len);
		    else
			    hipLaunchKernelGGL(reorder_kernel<16>, grid, dim3(256), 0, stream(), l, c, slot, parent, n_beams, since, len);
	    }))
		return rc;
	return ok();
}

int hako_gpu_tree_plan(const int *slot, const int *base, const int *parent, int n_seq, int n_tree, uint64_t *seen,
                       int *node_slot, int *row, int *turn) {
	if (int rc = tree_check(n_seq, n_tree)) return rc;
	if (n_seq && (!base || !parent)) return set_error(HAKO_GPU_EINVAL, "null bases or parents");
	if ((uintptr_t)seen & 7) return set_error(HAKO_GPU_EINVAL, "masks are not 8-byte aligned");
	if (int rc = require_device()) return rc;
	if (n_seq == 0) return ok();
	hipLaunchKernelGGL(tree_plan_kernel, dim3((n_seq + kTreeWaves - 1) / kTreeWaves), dim3(64 * kTreeWaves), 0, stream(), slot, base, parent,
	                   n_seq, n_tree, seen, node_slot, row, turn);
	HK_LAUNCHED("tree plan");
	return ok();
}

int hako_gpu_tree_accept(const int *parent, const int *token, const int *pick, const int *base, int n_seq, int n_tree,
                         int *path, int *n_path, int *next, int *new_base) {
	if (int rc = tree_check(n_seq, n_tree)) return rc;
	if (n_seq && (!parent || !token || !pick || !path || !n_path || !next)) return set_error(HAKO_GPU_EINVAL, "null argument");
	if (!base != !new_base) return set_error(HAKO_GPU_EINVAL, "one of base and new_base is null");
	if (int rc = require_device()) return rc;
	if (n_seq == 0) return ok();
	hipLaunchKernelGGL(tree_accept_kernel, dim3((n_seq + kTreeWaves - 1) / kTreeWaves), dim3(64 * kTreeWaves), 0, stream(), parent, token,
	                   pick, base, n_seq, n_tree, path, n_path, next, new_base);
	HK_LAUNCHED("tree path");
	return ok();
}

int hako_gpu_kv_keep(const hako_gpu_kv *kv, int n_kv, const int *slot, const int *base, const int *path,
                     const int *n_path, int n_seq, int n_tree) {
	if (int rc = caches_check(kv, n_kv)) return rc;
	if (int rc = tree_check(n_seq, n_tree)) return rc;
	if (n_seq > 65535) return set_error(HAKO_GPU_EINVAL, "%d sequences in one call (at most 65535)", n_seq);
	if (n_seq && (!base || !path || !n_path)) return set_error(HAKO_GPU_EINVAL, "null bases or paths");
	if (!slot && n_seq > kv->n_slots)
		return set_error(HAKO_GPU_EINVAL, "%d sequences without slots in a cache of %d", n_seq, kv->n_slots);
	if (int rc = require_device()) return rc;
	if (n_seq == 0) return ok();
	const Shape c = shape_of(kv);
	if (int rc = heads_check(n_kv, c, n_seq)) return rc;
	if (int rc = each_layers(kv, n_kv, [&](const Layers &l, int n) {
		    const int64_t waves = (int64_t)n * c.kvh * 2;
		    hipLaunchKernelGGL(keep_kernel, dim3((unsigned)((waves + kKeepWaves - 1) / kKeepWaves), n_seq), dim3(64 * kKeepWaves), 0, stream(), l, c,
		                       n, slot, base, path, n_path, n_tree);
	    }))
		return rc;
	return ok();
}

}  // extern "C"
