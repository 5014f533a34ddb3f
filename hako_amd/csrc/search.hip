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
// register 4 i + c; equal ones rank by position. Of a tile only what may still
// be among the n best is looked at one by one: values above the n-th best so
// far, and where more than n lanes have such values, above the n-th largest of
// the lanes' own maxima (found bit by bit, a ballot each), which at most n - 1
// lanes exceed. So no tile has more than n (E + 1) candidates, whatever the
// values are, and an ordinary one has about n at first and hardly any later.
// Candidates and the list so far rank each other in LDS.
template <int E>
struct Best {
	struct Lds {
		float v[HAKO_MAX_PICK * (E + 2)], lv[HAKO_MAX_PICK];
		int i[HAKO_MAX_PICK * (E + 2)], li[HAKO_MAX_PICK];   // li, lv: the list, best first
	};
	int n, count;   // wanted, in the list
	float least;    // a later value has to be larger

	__device__ __forceinline__ void start(int want) {
		n = want;
		count = 0;
		least = -kInf;
	}

	__device__ __forceinline__ void tile(const float (&x)[E], int pos0, Lds &s, int lane) {
		float mx = -kInf;
#pragma unroll
		for (int e = 0; e < E; e++) mx = __builtin_fmaxf(mx, x[e]);
		const uint64_t hits = __ballot(mx > least);
		if (!hits) return;
		float t = least;
		int ties = 0;   // values equal to t that may come in, the first ones
		if (__popcll(hits) > n) {
			const uint32_t b = __builtin_bit_cast(uint32_t, mx), key = b >> 31 ? ~b : b | 0x80000000u;
			uint32_t k = 0;
			for (int bit = 31; bit >= 0; bit--) {
				const uint32_t up = k | 1u << bit;
				k = __popcll(__ballot(key >= up)) >= n ? up : k;
			}
			t = __builtin_bit_cast(float, k >> 31 ? k & 0x7FFFFFFFu : ~k);
			ties = n;
		}
		int c = count;
		if (lane < count) {
			s.v[lane] = s.lv[lane];
			s.i[lane] = s.li[lane];
		}
#pragma unroll
		for (int e = 0; e < E; e++) {
			const uint64_t m = __ballot(x[e] > t);
			if (!m) continue;
			if (x[e] > t) {
				const int at = c + lanes_below(m);
				s.v[at] = x[e];
				s.i[at] = pos0 + ((e >> 2) * 64 + lane) * 4 + (e & 3);
			}
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
						if (before < ties) {
							s.v[c + before] = t;
							s.i[c + before] = pos0 + ((g >> 2) * 64 + lane) * 4 + e;
						}
						before++;
					}
				c += min(all, ties);
				ties -= all;
			}
		}
		wave_sync();
		for (int j = lane; j < c; j += 64) {
			const float v = s.v[j];
			const int i = s.i[j];
			int rank = 0;
			for (int k = 0; k < c; k++) rank += s.v[k] > v || (s.v[k] == v && s.i[k] < i);
			if (rank < n) {
				s.lv[rank] = v;
				s.li[rank] = i;
			}
		}
		wave_sync();
		count = min(c, n);
		if (count == n) least = s.lv[n - 1];
	}
};

// ── beam selection ──
//
// Two launches: waves over parts of the rows, then a workgroup a request.
// exp sums are taken against the part's maximum, in fp32 with the argument's
// rounding put right, four at a time into 64 bits, and meet in 64 bits.
constexpr int kPickE = 16;                 // values of a lane's tile
constexpr int kPickTile = 64 * kPickE;
constexpr int kPickWaves = 4;

// Per row and part: the largest value, the sum of exp(x - it), n_pick values
// and their tokens, best first, -inf where there are fewer.
struct Parts {
	double *sum;
	float *top, *v;
	int *i;
};

__device__ __forceinline__ float exp_(float d) {   // exp(d), d <= 0; NaN stays NaN
	d = d < -104.0f ? -104.0f : d;   // (0 from there on, -inf among them)
	const float t = d * 1.44269502f;
	const float r = __builtin_fmaf(d, 1.44269502f, -t) + d * 1.925963e-8f;   // log2(e) d - t
	const float e = __builtin_amdgcn_exp2f(t);
	return __builtin_fmaf(e, r * 0.693147180f, e);
}

__global__ __launch_bounds__(64 * kPickWaves) void beam_part_kernel(const float *__restrict__ logits, int64_t ld, int vocab,
                                                                    const int *__restrict__ done, int parts, int span,
                                                                    int n_pick, Parts out) {
	__shared__ typename Best<kPickE>::Lds lds[kPickWaves];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int part = blockIdx.x * kPickWaves + wave;
	const int64_t row = blockIdx.y;
	if (part >= parts || (done && done[row])) return;
	const int from = part * span, to = min(vocab, from + span);
	const float *src = logits + row * ld + from;
	const __amdgpu_buffer_rsrc_t r = stream_rsrc(uniform_ptr(src), (uint32_t)(to - from) * 4u);
	Best<kPickE> best;
	best.start(n_pick);
	float top = -kInf;
	double sum = 0.0;
	bool bad = false;
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
		if (t + kPickTile > to - from) {
#pragma unroll
			for (int e = 0; e < kPickE; e++) z[e] = t + ((e >> 2) * 64 + lane) * 4 + (e & 3) < to - from ? z[e] : -kInf;
		}
		float mx = -kInf;
#pragma unroll
		for (int e = 0; e < kPickE; e++) mx = __builtin_fmaxf(mx, z[e]);
		mx = wave_max(mx);
		if (mx > top) {
			sum *= exp((double)top - (double)mx);
			top = mx;
		}
		if (top > -kInf) {
#pragma unroll
			for (int e = 0; e < kPickE; e += 4)
				sum += (double)((exp_(z[e] - top) + exp_(z[e + 1] - top)) + (exp_(z[e + 2] - top) + exp_(z[e + 3] - top)));
		} else {
#pragma unroll
			for (int e = 0; e < kPickE; e++) bad |= z[e] != z[e];
		}
		best.tile(z, from + t, lds[wave], lane);
	};
	const int n = to - from;
	load(x, 0);
	for (int t = 0; t < n; t += 2 * kPickTile) {
		if (t + kPickTile < n) load(y, t + kPickTile);
		use(x, t);
		if (t + kPickTile >= n) break;
		if (t + 2 * kPickTile < n) load(x, t + 2 * kPickTile);
		use(y, t + kPickTile);
	}
#pragma unroll
	for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k);
	if (__any(bad)) sum = __builtin_nan("");
	const int64_t rec = row * parts + part;
	if (lane == 0) {
		out.top[rec] = top;
		out.sum[rec] = sum;
	}
	if (lane < n_pick) {
		out.v[rec * n_pick + lane] = lane < best.count ? lds[wave].lv[lane] : -kInf;
		out.i[rec * n_pick + lane] = lane < best.count ? lds[wave].li[lane] : -1;
	}
}

constexpr int kJoinE = 4;

// A wave a beam: its sum and its n_pick best; then the request's best of those.
__global__ __launch_bounds__(64 * HAKO_MAX_BEAMS) void beam_join_kernel(const float *__restrict__ score, const int *__restrict__ done,
                                                                        int eos, int n_beams, int n_pick, int parts, int arrange,
                                                                        Parts in, int *__restrict__ parent, int *__restrict__ token,
                                                                        float *__restrict__ score_out, int *__restrict__ done_out) {
	__shared__ typename Best<kJoinE>::Lds lds[HAKO_MAX_BEAMS];
	__shared__ double val[HAKO_MAX_BEAMS * HAKO_MAX_PICK];
	__shared__ int tok[HAKO_MAX_BEAMS * HAKO_MAX_PICK], pick[HAKO_MAX_PICK];
	const int lane = threadIdx.x & 63, b = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int64_t req = blockIdx.x, row = req * n_beams + b;
	const double old = (double)score[row];
	if (threadIdx.x < HAKO_MAX_PICK) pick[threadIdx.x] = -1;
	if (done && done[row]) {
		if (lane < n_pick) {
			val[b * n_pick + lane] = lane == 0 ? old : -(double)kInf;
			tok[b * n_pick + lane] = eos;
		}
	} else {
		const int64_t rec = row * parts;
		float top = -kInf;
		for (int p = lane; p < parts; p += 64) top = __builtin_fmaxf(top, in.top[rec + p]);
		top = wave_max(top);
		double sum = 0.0;
		for (int p = lane; p < parts; p += 64) {
			const float t = in.top[rec + p];
			sum += t == -kInf ? in.sum[rec + p] : in.sum[rec + p] * exp((double)t - (double)top);
		}
#pragma unroll
		for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k);
		const double lse = (double)top + log(sum);
		// the parts' lists in the order of their tokens; in a list equal values are in that order too
		Best<kJoinE> best;
		best.start(n_pick);
		const int n = parts * n_pick;
		for (int t = 0; t < n; t += 64 * kJoinE) {
			float x[kJoinE];
#pragma unroll
			for (int e = 0; e < kJoinE; e++) {
				const int at = t + lane * 4 + e;
				x[e] = at < n ? in.v[rec * n_pick + at] : -kInf;
			}
			best.tile(x, t, lds[b], lane);
		}
		if (lane < n_pick) {
			const bool on = lane < best.count;
			val[b * n_pick + lane] = on ? old + ((double)lds[b].lv[lane] - lse) : -(double)kInf;
			tok[b * n_pick + lane] = on ? in.i[rec * n_pick + lds[b].li[lane]] : -1;
		}
	}
	__syncthreads();
	// a beam's list falls, so that the place in it stands for logits and tokens
	const int n = n_beams * n_pick;
	for (int f = threadIdx.x; f < n; f += blockDim.x) {
		const double v = val[f];
		if (!(v > -(double)kInf)) continue;
		int rank = 0;
		for (int g = 0; g < n; g++) rank += val[g] > v || (val[g] == v && g < f);
		if (rank < n_pick) pick[rank] = f;
	}
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
	if (done_out) done_out[o] = f >= 0 && (t == eos || (done && done[req * n_beams + from]));
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
// map of places is good.
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
		uint4 x[B];
#pragma unroll
		for (int b = 0; b < B; b++)
			if (src[b] >= 0) x[b] = *(const uint4 *)(codes + src[b] * c.row + 16 * (first + u));
#pragma unroll
		for (int b = 0; b < B; b++)
			if (src[b] >= 0) *(uint4 *)(codes + dst[b] * c.row + 16 * (first + u)) = x[b];
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
// then its stores, so that a row may be another one's place.
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
		if (i * 64 >= rows * units) break;
		const int u = i * 64 + lane, d = u >> lg, f = __shfl(from, d & 63);
		if (d < rows && f >= 0) x[i] = *(const uint4 *)(codes + (int64_t)f * c.row + 16 * (u & (units - 1)));
	}
	// every load's data is here before the first store
	asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
	if (from >= 0) scales[lane] = y;
#pragma unroll
	for (int i = 0; i < 16; i++) {
		if (i * 64 >= rows * units) break;
		const int u = i * 64 + lane, d = u >> lg, f = __shfl(from, d & 63);
		if (d < rows && f >= 0) *(uint4 *)(codes + (int64_t)d * c.row + 16 * (u & (units - 1))) = x[i];
	}
}

// ── drafted trees: a wave a tree, a lane a node ──

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
	if (row) row[at] = on ? b + lane : -1;
	if (turn) turn[at] = on ? b + __popcll(m) - 1 : -1;
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

// Workgroups of a launch over the heads of its caches, each with n sequences' rows, some to spare.
int heads_check(int n_kv, const Shape &c, int n) {
	const int64_t heads = (int64_t)(n_kv < kLayers ? n_kv : kLayers) * c.kvh * 2 * n;
	if (heads > kMaxThreads / 512) return set_error(HAKO_GPU_EINVAL, "%lld heads of %d sequences in one call", (long long)heads, n);
	return HAKO_GPU_OK;
}

}  // namespace

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
	// parts of whole tiles, until the waves fill the chip
	const int tiles = (vocab + kPickTile - 1) / kPickTile, want = (8 * cu_count() + rows - 1) / rows;
	const int span = (tiles + want - 1) / want * kPickTile, parts = (vocab + span - 1) / span;
	const size_t recs = (size_t)rows * parts;
	void *p = nullptr;
	if (int rc = workspace(kWsSearch, recs * (12 + 8 * (size_t)n_pick), &p)) return rc;
	Parts out;
	out.sum = (double *)p;
	out.top = (float *)(out.sum + recs);
	out.v = out.top + recs;
	out.i = (int *)(out.v + recs * n_pick);
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
		    const int64_t most = ((int64_t)c.max_seq * (c.row / 16) + 255) / 256, fill = 8 * cu_count() / (heads * n_req) + 1;
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
