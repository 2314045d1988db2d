// Token log-probabilities and the losses over them: paired preferences and clipped policy updates, each with its gradient to the logits.
//
//   row r = a T + t (sequence a, position t) counts if it is not padded and its target lies in [0, V)
//   log-probability  lp = x_t - m - log(s), m = max_v x_v, s = sum_v exp(x_v - m);   d lp / d x_v = [v = target] - exp(x_v - m) / s
//   preference       u_a = sum_t (lp - ref) over a's counted rows, pair i = sequences (i, n + i), z = beta (u_i - u_{n+i}), loss = sum_i w_i l(z_i) / sum_i w_i,
//                    l = -(1 - e) log sigmoid(z) - e log sigmoid(-z)  |  max(0, 1 - z)  |  (z / beta - 1 / (2 beta))^2
//   policy           q = exp(lp - old), l = -min(q a, clip(q, 1 - lo, 1 + hi) a) + k (exp(d) - d - 1), d = ref - lp;  loss = mean over counted rows, or over sequences of
//                    the mean over a sequence's counted rows
//
// HBM-bound: V logits a row in, V gradients a row out.  A row belongs to a workgroup that holds it in registers between the sum and the gradient; padded rows are not read.
// The exponentials and the sums over the vocabulary are fp32; a log-probability is formed and added up over its sequence in fp64 (a handful of operations a ROW):
// the losses take differences of sums that nearly cancel.
#include "novic_hip.h"
#include "rowvec.hpp"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct Rows {
	const void* logits;
	long long ldl;
	void* dlogits;
	long long ldd;
	const void* target;
	const uint8_t* pad;
	long long ldt, ldp;  // of target and pad, in elements
	int tok_bytes, A, T, V;
};

__device__ __forceinline__ int counted_target(const Rows& g, int a, int t) {  // -1: the position does not count
	if (g.pad && g.pad[a * g.ldp + t]) return -1;
	const long long v = g.tok_bytes == 8 ? ((const long long*)g.target)[a * g.ldt + t] : (long long)((const int*)g.target)[a * g.ldt + t];
	return v < 0 || v >= g.V ? -1 : (int)v;
}

// Workgroup -> row.  A grid's extent in threads is 32 bits, so rows beyond 2^20 go to its second dimension.
__device__ __forceinline__ int row_index(const Rows& g) {
	const long long r = (long long)blockIdx.y * gridDim.x + blockIdx.x;
	return r < (long long)g.A * g.T ? (int)r : -1;
}

// log(s) to 1e-16 relative of a sum in [1, 2^31] without the cost of a double-precision logarithm: s = 2^k f, f in [0.7, 1.42): |logf(f)| < 0.36, its rounding 3e-8 absolute
__device__ __forceinline__ double log_wide(float s) {
	int k;
	float f = frexpf(s, &k);
	if (f < 0.70710678f) {
		f += f;
		--k;
	}
	return fma((double)k, 0.69314718055994530942, (double)logf(f));
}

// reductions over a workgroup of THREADS; `red` has a slot per wave; ends with everyone holding the value and `red` free again after the next barrier of the caller
template <int THREADS>
__device__ __forceinline__ float block_max(float v, float* red) {
	v = wave_max(v);
	if constexpr (THREADS > 64) {
		if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
		__syncthreads();
		constexpr int W = THREADS / 64;
		v = red[threadIdx.x & (W - 1)];
#pragma unroll
		for (int o = W / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
	}
	return v;
}
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* red) {
	v = wave_sum(v);
	if constexpr (THREADS > 64) {
		if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
		__syncthreads();
		v = team_sum<THREADS / 64>(red[threadIdx.x & (THREADS / 64 - 1)]);
	}
	return v;
}

// A row in registers.  x[] becomes exp(x - m) in sum(); elements that another lane owns too are zeros there.
template <typename T, int CH, int THREADS, int NC>
struct RowTile {
	float x[NC][CH];
	float m, s;
	__device__ __forceinline__ static int own(int c) { return (c * THREADS + (int)threadIdx.x) * CH; }
	__device__ __forceinline__ static int at(int c, int V) { return min(own(c), V - CH); }
	__device__ __forceinline__ void load(const T* row, int V) {
		RawVec<T, CH> raw[NC];
#pragma unroll
		for (int c = 0; c < NC; ++c)
			if (c * THREADS * CH < V) raw[c] = load_vec<T, CH>(elem(row, at(c, V)));
#pragma unroll
		for (int c = 0; c < NC; ++c)
#pragma unroll
			for (int i = 0; i < CH; ++i) x[c][i] = c * THREADS * CH < V ? raw[c].get(i) : -INFINITY;
	}
	__device__ __forceinline__ void sum(int V, float* red) {
		float t = -INFINITY;
#pragma unroll
		for (int c = 0; c < NC; ++c)
#pragma unroll
			for (int i = 0; i < CH; ++i) t = fmaxf(t, x[c][i]);
		m = block_max<THREADS>(t, red);
		t = 0.f;
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			if (c * THREADS * CH >= V) {
#pragma unroll
				for (int i = 0; i < CH; ++i) x[c][i] = 0.f;
				continue;
			}
#pragma unroll
			for (int i = 0; i < CH; ++i) {
				x[c][i] = __builtin_amdgcn_exp2f((x[c][i] - m) * LOG2E);
				if ((c + 1) * THREADS * CH > V && at(c, V) + i < own(c)) x[c][i] = 0.f;
				t += x[c][i];
			}
		}
		s = block_sum<THREADS>(t, red + THREADS / 64);
	}
	// dlogits = g ([v = target] - x / s)
	__device__ __forceinline__ void grad(T* row, int V, int target, float g) {
		const float k = -g / s;
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			if (own(c) >= V) continue;
			float o[CH];
			const int es = at(c, V);
#pragma unroll
			for (int i = 0; i < CH; ++i) o[i] = (k * x[c][i] + (es + i == target ? g : 0.f));
			store_own<T, CH>(row, es, own(c), o);
		}
	}
};

template <typename T, int CH, int THREADS>
__device__ __forceinline__ void zero_row(T* row, int V) {
	float o[CH];
#pragma unroll
	for (int i = 0; i < CH; ++i) o[i] = 0.f;
	for (int e0 = threadIdx.x * CH; e0 < V; e0 += THREADS * CH) store_own<T, CH>(row, min(e0, V - CH), e0, o);
}

// ---- log-probabilities -------------------------------------------------------------------------------------------------------------------------------------------
struct LogpOut {
	float* logp;       // [A][T] or null
	float* lse;        // [A T] or null: m + log(s)
	const float* ref;  // [A][T] or null
	double* diff;      // [A T] or null: lp - ref, 0 where the row does not count
	float2* norm;      // [A T] or null: (m, 1 / s)
	long long ldo, ldref;
};
__device__ __forceinline__ void put_logp(const LogpOut& o, int r, int a, int t, bool counts, double lp, float m, float s) {
	if (o.logp) o.logp[a * o.ldo + t] = counts ? (float)lp : 0.f;
	if (o.lse) o.lse[r] = counts ? (float)((double)m + log_wide(s)) : 0.f;
	if (o.diff) o.diff[r] = counts ? lp - (double)o.ref[a * o.ldref + t] : 0.0;
	if (o.norm) o.norm[r] = counts ? make_float2(m, 1.f / s) : make_float2(0.f, 0.f);
}

template <typename T, int CH, int THREADS, int NC>
__global__ __launch_bounds__(THREADS) void logp_kernel(const Rows g, const LogpOut o) {
	__shared__ float red[2 * THREADS / 64];
	const int r = row_index(g);
	if (r < 0) return;
	const int a = r / g.T, t = r - a * g.T;
	const int target = counted_target(g, a, t);
	if (target < 0) {
		if (threadIdx.x == 0) put_logp(o, r, a, t, false, 0.0, 0.f, 1.f);
		return;
	}
	const T* row = (const T*)g.logits + (long long)r * g.ldl;
	RowTile<T, CH, THREADS, NC> tile;
	tile.load(row, g.V);
	const float xt = (float)row[target];
	tile.sum(g.V, red);
	if (threadIdx.x == 0) put_logp(o, r, a, t, true, ((double)xt - (double)tile.m) - log_wide(tile.s), tile.m, tile.s);
}

// rows beyond the register forms: maximum and sum in one pass with a running maximum
template <typename T, int CH, int THREADS>
__device__ __forceinline__ void long_row_sum(const T* row, int V, float* red, float& m, float& s) {
	float tm = -INFINITY, ts = 0.f;
	for (int e0 = threadIdx.x * CH; e0 < V; e0 += THREADS * CH) {
		const int es = min(e0, V - CH);
		const RawVec<T, CH> raw = load_vec<T, CH>(elem(row, es));
		float top = tm;
#pragma unroll
		for (int i = 0; i < CH; ++i) top = fmaxf(top, raw.get(i));
		const float base = top == -INFINITY ? 0.f : top;  // (nothing but -inf yet: their exponentials are zeros)
		ts *= __builtin_amdgcn_exp2f((tm - base) * LOG2E);
#pragma unroll
		for (int i = 0; i < CH; ++i) ts += es + i >= e0 ? __builtin_amdgcn_exp2f((raw.get(i) - base) * LOG2E) : 0.f;
		tm = top;
	}
	m = block_max<THREADS>(tm, red);
	const float base = m == -INFINITY ? 0.f : m;
	s = block_sum<THREADS>(ts * __builtin_amdgcn_exp2f(((tm == -INFINITY ? base : tm) - base) * LOG2E), red + THREADS / 64);
}
template <typename T, int CH, int THREADS>
__global__ __launch_bounds__(THREADS) void logp_long_kernel(const Rows g, const LogpOut o) {
	__shared__ float red[2 * THREADS / 64];
	const int r = row_index(g);
	if (r < 0) return;
	const int a = r / g.T, t = r - a * g.T;
	const int target = counted_target(g, a, t);
	if (target < 0) {
		if (threadIdx.x == 0) put_logp(o, r, a, t, false, 0.0, 0.f, 1.f);
		return;
	}
	const T* row = (const T*)g.logits + (long long)r * g.ldl;
	const float xt = (float)row[target];
	float m, s;
	long_row_sum<T, CH, THREADS>(row, g.V, red, m, s);
	if (threadIdx.x == 0) put_logp(o, r, a, t, true, ((double)xt - (double)m) - log_wide(s), m, s);
}

// ---- gradient of log-probabilities: dlogits = coef (1[v = target] - exp(x - m) / s) ----------------------------------------------------------------------------------
struct GradIn {
	const float* lse;     // [A T] (m + log s), or null:
	const float2* norm;   // [A T] (m, 1 / s)
	const float* grad;    // element (a, t) at grad[a * lda + t * ldt]
	long long lda, ldt;
	const float* scale;   // device scalar or null
};
template <typename T, int CH, int THREADS>
__global__ __launch_bounds__(THREADS) void logp_grad_kernel(const Rows g, const GradIn in) {
	const int r = row_index(g);
	if (r < 0) return;
	const int a = r / g.T, t = r - a * g.T;
	const int target = counted_target(g, a, t);
	T* out = (T*)g.dlogits + (long long)r * g.ldd;
	if (target < 0) {
		zero_row<T, CH, THREADS>(out, g.V);
		return;
	}
	const T* row = (const T*)g.logits + (long long)r * g.ldl;
	float coef = in.grad[a * in.lda + t * in.ldt];
	if (in.scale) coef *= *in.scale;
	float m, k = -coef;
	if (in.norm) {
		const float2 n = in.norm[r];
		m = n.x;
		k *= n.y;
	} else {
		m = in.lse[r];
	}
	for (int e0 = threadIdx.x * CH; e0 < g.V; e0 += THREADS * CH) {
		const int es = min(e0, g.V - CH);
		const RawVec<T, CH> raw = load_vec<T, CH>(elem(row, es));
		float o[CH];
#pragma unroll
		for (int i = 0; i < CH; ++i) o[i] = (k * __builtin_amdgcn_exp2f((raw.get(i) - m) * LOG2E) + (es + i == target ? coef : 0.f));
		store_own<T, CH>(out, es, e0, o);
	}
}

// ---- preference loss ---------------------------------------------------------------------------------------------------------------------------------------------
struct Pref {
	const double* diff;   // [2 n][T]
	const float* weight;  // [n] or null
	int n, T, kind;
	double beta, smoothing, grad_scale;
	float* margin;        // [n] or null
	float* coef;          // [2 n]: gradient of the loss to a sequence's u, times sum(w) until pref_finish_kernel has made the scale
	double* each;         // [2][n]: w l, w z
	float* scale;         // device scalar: grad_scale / sum(w)
	float* stats;         // [3]: loss, mean margin, sum(w)
};
__device__ __forceinline__ void pref_pair(const Pref& g, int i, double up, double un) {
	const double z = g.beta * (up - un), w = g.weight ? (double)g.weight[i] : 1.0;
	double l, dz;
	if (g.kind == NOVIC_PREF_SIGMOID) {
		const double soft = log1p(exp(-fabs(z)));  // -log sigmoid(z) = soft + max(-z, 0)
		l = (1.0 - g.smoothing) * (soft + fmax(-z, 0.0)) + g.smoothing * (soft + fmax(z, 0.0));
		dz = 1.0 / (1.0 + exp(-z)) - (1.0 - g.smoothing);
	} else if (g.kind == NOVIC_PREF_HINGE) {
		l = z < 1.0 ? 1.0 - z : (z >= 1.0 ? 0.0 : z);  // (a NaN stays one)
		dz = z < 1.0 ? -1.0 : (z >= 1.0 ? 0.0 : z);
	} else {
		const double u = (z - 0.5) / g.beta;
		l = u * u;
		dz = 2.0 * u / g.beta;
	}
	if (g.margin) g.margin[i] = (float)z;
	const float c = (float)(w * dz * g.beta);
	g.coef[i] = c;
	g.coef[g.n + i] = -c;
	g.each[i] = w * l;
	g.each[g.n + i] = w * z;
}
// sum of one sequence's T values by `lanes` consecutive lanes (a power of two up to 64), in a fixed order
__device__ __forceinline__ double seq_sum(const double* v, int T, int lane, int lanes) {
	double u = 0.0;
	for (int t = lane; t < T; t += lanes) u += v[t];
	for (int o = lanes / 2; o > 0; o >>= 1) u += __shfl_xor(u, o, 64);
	return u;
}
__global__ __launch_bounds__(256) void pref_pair_kernel(const Pref g, int lanes) {
	const long long id = ((long long)blockIdx.x * 256 + threadIdx.x) / lanes;
	const int lane = threadIdx.x % lanes;
	if (id >= g.n) return;
	const int i = (int)id;
	const double up = seq_sum(g.diff + (long long)i * g.T, g.T, lane, lanes), un = seq_sum(g.diff + ((long long)g.n + i) * g.T, g.T, lane, lanes);
	if (lane == 0) pref_pair(g, i, up, un);
}
// three sums over a workgroup of 1024 in a fixed order; thread 0 has them
__device__ __forceinline__ void sum3_1024(double& a, double& b, double& c, double* red) {
#pragma unroll
	for (int o = 32; o > 0; o >>= 1) {
		a += __shfl_xor(a, o, 64);
		b += __shfl_xor(b, o, 64);
		c += __shfl_xor(c, o, 64);
	}
	const int w = threadIdx.x >> 6;
	if ((threadIdx.x & 63) == 0) {
		red[w] = a;
		red[16 + w] = b;
		red[32 + w] = c;
	}
	__syncthreads();
	if (threadIdx.x == 0) {
		a = b = c = 0.0;
		for (int i = 0; i < 16; ++i) {
			a += red[i];
			b += red[16 + i];
			c += red[32 + i];
		}
	}
}
__global__ __launch_bounds__(1024) void pref_finish_kernel(const Pref g) {
	__shared__ double red[48];
	double l = 0.0, z = 0.0, w = 0.0;
	for (int i = threadIdx.x; i < g.n; i += 1024) {
		l += g.each[i];
		z += g.each[g.n + i];
		w += g.weight ? (double)g.weight[i] : 1.0;
	}
	sum3_1024(l, z, w, red);
	if (threadIdx.x == 0) {
		const bool any = w != 0.0;  // (no weight at all: no loss and no gradient)
		g.stats[0] = any ? (float)(l / w) : 0.f;
		g.stats[1] = any ? (float)(z / w) : 0.f;
		g.stats[2] = (float)w;
		*g.scale = any ? (float)(g.grad_scale / w) : 0.f;
	}
}

// ---- policy loss -------------------------------------------------------------------------------------------------------------------------------------------------
struct Policy {
	const float *old, *adv, *ref;  // old, ref [A][T]; adv at adv[a * lda + t * ldt]
	long long ldold, ldref, lda, ldt;
	float lo, hi, kl_coef, grad_scale;
	int per_seq;
	float* logp;       // [A][T] or null
	long long ldo;
	int* len;          // [A]: counted rows of a sequence
	int* part;         // [2][parts]: counted rows, sequences with any, of the sequences of one block of policy_count_kernel
	int parts;
	float* each;       // [3][A T]: loss, KL, clipped, each times the row's share of the mean
	float* stats;      // [4]: loss, mean KL, clipped share, counted rows
};
__global__ __launch_bounds__(256) void policy_count_kernel(const Rows g, const Policy p, int lanes) {
	__shared__ int red[8];
	const int lane = threadIdx.x % lanes, teams = 256 / lanes;
	int rows = 0, seqs = 0;
	for (int a = blockIdx.x * teams + threadIdx.x / lanes; a < g.A; a += gridDim.x * teams) {
		int n = 0;
		for (int t = lane; t < g.T; t += lanes) n += counted_target(g, a, t) >= 0;
		for (int o = lanes / 2; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
		if (lane == 0) {
			p.len[a] = n;
			rows += n;
			seqs += n > 0;
		}
	}
#pragma unroll
	for (int o = 32; o > 0; o >>= 1) {
		rows += __shfl_xor(rows, o, 64);
		seqs += __shfl_xor(seqs, o, 64);
	}
	if ((threadIdx.x & 63) == 0) {
		red[threadIdx.x >> 6] = rows;
		red[4 + (threadIdx.x >> 6)] = seqs;
	}
	__syncthreads();
	if (threadIdx.x < 2) p.part[threadIdx.x * p.parts + blockIdx.x] = red[4 * threadIdx.x] + red[4 * threadIdx.x + 1] + red[4 * threadIdx.x + 2] + red[4 * threadIdx.x + 3];
}
// the counts of all blocks, by one wave (at most 64 parts)
__device__ __forceinline__ int policy_total(const Policy& p, int which) {
	const int lane = threadIdx.x & 63;
	int n = lane < p.parts ? p.part[which * p.parts + lane] : 0;
#pragma unroll
	for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
	return n;
}
// The gradient of the whole loss to a row's log-probability.  The ratio and the KL term are exponentials of small differences that were formed in fp64.
struct PolicyRow {
	float q, held, adv;
	double d;
	bool whole;  // the unclipped side of the minimum (a NaN takes it and stays one)
};
__device__ __forceinline__ float policy_grad(const Policy& p, int a, int t, double lp, float share, PolicyRow& w) {
	w.q = expf((float)(lp - (double)p.old[a * p.ldold + t]));
	w.adv = p.adv[a * p.lda + t * p.ldt];
	w.held = fminf(fmaxf(w.q, 1.f - p.lo), 1.f + p.hi);
	w.whole = !(w.q * w.adv > w.held * w.adv);
	float g = w.whole ? -w.q * w.adv : 0.f;
	w.d = 0.0;
	if (p.ref) {
		w.d = (double)p.ref[a * p.ldref + t] - lp;
		g -= p.kl_coef * expm1f((float)w.d);
	}
	return g * share * p.grad_scale;
}
__device__ __forceinline__ float policy_share(const Rows& g, const Policy& p, int a) {
	return p.per_seq ? 1.f / ((float)p.len[a] * (float)policy_total(p, 1)) : 1.f / (float)policy_total(p, 0);
}
// what one thread of the row writes: its log-probability and its terms of the means
__device__ __forceinline__ void policy_put(const Rows& g, const Policy& p, int r, int a, int t, double lp, float share, const PolicyRow& w) {
	const long long R = (long long)g.A * g.T;
	const double kl = p.ref ? expm1(w.d) - w.d : 0.0;
	if (p.logp) p.logp[a * p.ldo + t] = (float)lp;
	p.each[r] = (float)(((w.whole ? -(double)w.q * w.adv : -(double)w.held * w.adv) + (double)p.kl_coef * kl) * share);
	p.each[R + r] = (float)(kl * share);
	p.each[2 * R + r] = w.whole ? 0.f : share;
}
__device__ __forceinline__ void policy_put_none(const Rows& g, const Policy& p, int r, int a, int t) {
	const long long R = (long long)g.A * g.T;
	if (p.logp) p.logp[a * p.ldo + t] = 0.f;
	p.each[r] = p.each[R + r] = p.each[2 * R + r] = 0.f;
}
template <typename T, int CH, int THREADS, int NC>
__global__ __launch_bounds__(THREADS) void policy_kernel(const Rows g, const Policy p) {
	__shared__ float red[2 * THREADS / 64];
	const int r = row_index(g);
	if (r < 0) return;
	const int a = r / g.T, t = r - a * g.T;
	const int target = counted_target(g, a, t);
	T* out = (T*)g.dlogits + (long long)r * g.ldd;
	if (target < 0) {
		if (g.dlogits) zero_row<T, CH, THREADS>(out, g.V);
		if (threadIdx.x == 0) policy_put_none(g, p, r, a, t);
		return;
	}
	const T* row = (const T*)g.logits + (long long)r * g.ldl;
	RowTile<T, CH, THREADS, NC> tile;
	tile.load(row, g.V);
	const float xt = (float)row[target], share = policy_share(g, p, a);
	tile.sum(g.V, red);
	const double lp = ((double)xt - (double)tile.m) - log_wide(tile.s);
	PolicyRow w;
	const float coef = policy_grad(p, a, t, lp, share, w);
	if (threadIdx.x == 0) policy_put(g, p, r, a, t, lp, share, w);
	if (g.dlogits) tile.grad(out, g.V, target, coef);
}
template <typename T, int CH, int THREADS>
__global__ __launch_bounds__(THREADS) void policy_long_kernel(const Rows g, const Policy p) {
	__shared__ float red[2 * THREADS / 64];
	const int r = row_index(g);
	if (r < 0) return;
	const int a = r / g.T, t = r - a * g.T;
	const int target = counted_target(g, a, t);
	T* out = (T*)g.dlogits + (long long)r * g.ldd;
	if (target < 0) {
		if (g.dlogits) zero_row<T, CH, THREADS>(out, g.V);
		if (threadIdx.x == 0) policy_put_none(g, p, r, a, t);
		return;
	}
	const T* row = (const T*)g.logits + (long long)r * g.ldl;
	const float xt = (float)row[target], share = policy_share(g, p, a);
	float m, s;
	long_row_sum<T, CH, THREADS>(row, g.V, red, m, s);
	const double lp = ((double)xt - (double)m) - log_wide(s);
	PolicyRow w;
	const float coef = policy_grad(p, a, t, lp, share, w);
	if (threadIdx.x == 0) policy_put(g, p, r, a, t, lp, share, w);
	if (!g.dlogits) return;
	const float k = -coef / s;
	for (int e0 = threadIdx.x * CH; e0 < g.V; e0 += THREADS * CH) {
		const int es = min(e0, g.V - CH);
		const RawVec<T, CH> raw = load_vec<T, CH>(elem(row, es));
		float o[CH];
#pragma unroll
		for (int i = 0; i < CH; ++i) o[i] = (k * __builtin_amdgcn_exp2f((raw.get(i) - m) * LOG2E) + (es + i == target ? coef : 0.f));
		store_own<T, CH>(out, es, e0, o);
	}
}
__global__ __launch_bounds__(1024) void policy_finish_kernel(const Rows g, const Policy p) {
	__shared__ double red[48];
	const long long R = (long long)g.A * g.T;
	double l = 0.0, k = 0.0, c = 0.0;
	for (long long r = threadIdx.x; r < R; r += 1024) {
		l += (double)p.each[r];
		k += (double)p.each[R + r];
		c += (double)p.each[2 * R + r];
	}
	sum3_1024(l, k, c, red);
	const int n = policy_total(p, 0);
	if (threadIdx.x == 0) {
		p.stats[0] = (float)l;
		p.stats[1] = (float)k;
		p.stats[2] = (float)c;
		p.stats[3] = (float)n;
	}
}

// ---- launches ----------------------------------------------------------------------------------------------------------------------------------------------------
// A register form holds threads * chunks vectors of CH elements; longer rows take the form that reads a row twice (its second pass comes out of L2 / the memory-side cache).
#define NOVIC_ROW_SHAPES(V, REG, LONG)                                                                     \
	if constexpr (CH == 1) { constexpr int TH = 64, NC = 1; REG; } /* fewer than eight columns */             \
	else if (V <= 64 * CH) { constexpr int TH = 64, NC = 1; REG; }                                           \
	else if (V <= 256 * CH) { constexpr int TH = 256, NC = 1; REG; }                                         \
	else if (V <= 512 * CH) { constexpr int TH = 256, NC = 2; REG; }                                         \
	else if (V <= 1024 * CH) { constexpr int TH = 256, NC = 4; REG; }                                        \
	else if (V <= 2048 * CH) { constexpr int TH = 256, NC = 8; REG; }                                        \
	else if (V <= 4096 * CH) { constexpr int TH = 1024, NC = 4; REG; }                                       \
	else if (V <= 8192 * CH) { constexpr int TH = 1024, NC = 8; REG; }                                       \
	else { constexpr int TH = 1024; LONG; }

dim3 rows_grid(const Rows& g) {
	const long long R = (long long)g.A * g.T, x = std::min<long long>(R, 1 << 20);
	return dim3((unsigned)x, (unsigned)((R + x - 1) / x));
}
template <typename T, int CH>
void launch_logp(const Rows& g, const LogpOut& o, hipStream_t stream) {
	const dim3 grid = rows_grid(g);
	NOVIC_ROW_SHAPES(g.V, (logp_kernel<T, CH, TH, NC><<<grid, dim3(TH), 0, stream>>>(g, o)),
	                 (logp_long_kernel<T, CH, TH><<<grid, dim3(TH), 0, stream>>>(g, o)))
}
template <typename T, int CH>
void launch_grad(const Rows& g, const GradIn& in, hipStream_t stream) {
	const dim3 grid = rows_grid(g);
	if (CH == 1 || g.V <= 64 * CH) logp_grad_kernel<T, CH, 64><<<grid, dim3(64), 0, stream>>>(g, in);
	else logp_grad_kernel<T, CH, 256><<<grid, dim3(256), 0, stream>>>(g, in);
}
template <typename T, int CH>
void launch_policy(const Rows& g, const Policy& p, hipStream_t stream) {
	const dim3 grid = rows_grid(g);
	NOVIC_ROW_SHAPES(g.V, (policy_kernel<T, CH, TH, NC><<<grid, dim3(TH), 0, stream>>>(g, p)),
	                 (policy_long_kernel<T, CH, TH><<<grid, dim3(TH), 0, stream>>>(g, p)))
}
#define NOVIC_ROW_TYPES(type, V, FN, ...)                                             \
	if (V < 8) NOVIC_TYPE_SWITCH(type, T, (FN<T, 1>(__VA_ARGS__)))                       \
	else if (type == NOVIC_TYPE_F32) FN<float, 4>(__VA_ARGS__);                          \
	else if (type == NOVIC_TYPE_BF16) FN<bf16, 8>(__VA_ARGS__);                          \
	else FN<f16, 8>(__VA_ARGS__);

const char* rows_bad(const Rows& g, int type) {
	if (type < NOVIC_TYPE_F32 || type > NOVIC_TYPE_F16) return "logits are fp32, bf16 or fp16";
	if (g.tok_bytes != 4 && g.tok_bytes != 8) return "tok_bytes must be 4 or 8";
	if (g.A < 0 || g.T < 0 || g.V < 1 || g.V > 1 << 28) return "A, T >= 0 and 1 <= V <= 2^28";
	const long long R = (long long)g.A * g.T;
	if (R >= (1LL << 31)) return "at most 2^31 - 1 token rows";
	if (R > 0 && (!g.logits || !g.target)) return "null pointer";
	if (R > 1 && (g.ldl < g.V || (g.dlogits && g.ldd < g.V))) return "leading dimensions >= V";
	if (g.A > 1 && (g.ldt < g.T || (g.pad && g.ldp < g.T))) return "leading dimensions of target and pad >= T";
	return nullptr;
}
Span logits_span(const Rows& g, int type) { return {g.logits, (long long)g.A * g.T, g.V * type_bytes(type), g.ldl * type_bytes(type)}; }
Span dlogits_span(const Rows& g, int type) { return {g.dlogits, (long long)g.A * g.T, g.V * type_bytes(type), g.ldd * type_bytes(type)}; }
Span target_span(const Rows& g) { return {g.target, g.A, (long long)g.T * g.tok_bytes, g.ldt * g.tok_bytes}; }
Span pad_span(const Rows& g) { return {g.pad, g.A, g.T, g.ldp}; }
Span token_span(const Rows& g, const float* p, long long ld) { return {p, g.A, 4LL * g.T, 4 * ld}; }  // fp32 [A][ld >= T]
Span vector_span(const void* p, long long bytes) { return {p, 1, bytes, 0}; }
int lanes_for(int T) {
	int lanes = 1;
	while (lanes < 64 && lanes * 4 < T) lanes *= 2;
	return lanes;
}
uint64_t up16(uint64_t n) { return (n + 15) / 16 * 16; }
constexpr int COUNT_PARTS = 64;
int count_parts(int A, int T) { return (int)std::min<long long>(COUNT_PARTS, ((long long)A * lanes_for(T) + 255) / 256); }

}  // namespace

extern "C" int novic_token_logprobs(const void* logits, int type, int64_t ldl, const void* target, int tok_bytes, int64_t ldt, const uint8_t* pad, int64_t ldp, int A, int T, int V,
                                    float* logp, int64_t ldo, float* lse, hipStream_t stream) {
	Rows g = {logits, ldl, nullptr, 0, target, pad, ldt, ldp, tok_bytes, A, T, V};
	const char* bad = rows_bad(g, type);
	NOVIC_CHECK(!bad, bad);
	if ((long long)A * T == 0) return 0;
	NOVIC_CHECK(logp && (A <= 1 || ldo >= T), "novic_token_logprobs: logp [A][ldo >= T]");
	NOVIC_APART("novic_token_logprobs", NOVIC_SPANS(token_span(g, logp, ldo), vector_span(lse, 4LL * A * T)), NOVIC_SPANS(target_span(g), pad_span(g), logits_span(g, type)), NOVIC_SPANS({}))
	LogpOut o = {};
	o.logp = logp; o.ldo = ldo; o.lse = lse;
	NOVIC_ROW_TYPES(type, V, launch_logp, g, o, stream)
	NOVIC_LAUNCH_CHECK();
	return 0;
}

extern "C" int novic_token_logprobs_bwd(const void* logits, int type, int64_t ldl, const void* target, int tok_bytes, int64_t ldt, const uint8_t* pad, int64_t ldp, int A, int T, int V,
                                        const float* lse, const float* grad, int64_t grad_lda, int64_t grad_ldt, void* dlogits, int64_t ldd, hipStream_t stream) {
	Rows g = {logits, ldl, dlogits, ldd, target, pad, ldt, ldp, tok_bytes, A, T, V};
	const char* bad = rows_bad(g, type);
	NOVIC_CHECK(!bad, bad);
	if ((long long)A * T == 0) return 0;
	NOVIC_CHECK(lse && grad && dlogits, "novic_token_logprobs_bwd: null pointer");
	NOVIC_CHECK(grad_ldt == 0 || grad_ldt == 1, "novic_token_logprobs_bwd: grad has unit stride along the positions, or one value a sequence");
	NOVIC_APART("novic_token_logprobs_bwd", NOVIC_SPANS(dlogits_span(g, type)),
	            NOVIC_SPANS(target_span(g), pad_span(g), vector_span(lse, 4LL * A * T), {grad, A, grad_ldt ? 4LL * T : 4, 4 * grad_lda}), NOVIC_SPANS(logits_span(g, type)))
	GradIn in = {};
	in.lse = lse; in.grad = grad; in.lda = grad_lda; in.ldt = grad_ldt;
	NOVIC_ROW_TYPES(type, V, launch_grad, g, in, stream)
	NOVIC_LAUNCH_CHECK();
	return 0;
}

// workspace: diff [2n T] fp64, each [2][n] fp64, norm [2n T] float2, coef [2n], scale
extern "C" uint64_t novic_preference_loss_ws(int n, int T) {
	if (n <= 0 || T <= 0) return 0;
	const uint64_t R = 2ull * n * T;
	return up16(8 * R) + up16(16ull * n) + up16(8 * R) + up16(8ull * n) + 16;
}
extern "C" int novic_preference_loss(const void* logits, int type, int64_t ldl, const void* target, int tok_bytes, int64_t ldt, const uint8_t* pad, int64_t ldp, int n, int T, int V,
                                     const float* ref, int64_t ldref, const float* weight, int kind, double beta, double smoothing, double grad_scale, float* logp, int64_t ldo,
                                     float* margin, void* dlogits, int64_t ldd, float* stats, void* ws, uint64_t ws_bytes, hipStream_t stream) {
	NOVIC_CHECK(n >= 1 && n <= (1 << 29) && T >= 1, "novic_preference_loss: at least one pair and one position");
	Rows g = {logits, ldl, dlogits, ldd, target, pad, ldt, ldp, tok_bytes, 2 * n, T, V};
	const char* bad = rows_bad(g, type);
	NOVIC_CHECK(!bad, bad);
	NOVIC_CHECK(ref && stats && ldref >= T && (!logp || ldo >= T), "novic_preference_loss: ref [2n][ldref >= T], stats [3]");
	NOVIC_CHECK(kind == NOVIC_PREF_SIGMOID || kind == NOVIC_PREF_HINGE || kind == NOVIC_PREF_SQUARE, "novic_preference_loss: unknown kind");
	NOVIC_CHECK(beta > 0.0 && smoothing >= 0.0 && smoothing < 0.5 && (smoothing == 0.0 || kind == NOVIC_PREF_SIGMOID), "novic_preference_loss: beta > 0; smoothing in [0, 0.5), with the sigmoid form only");
	NOVIC_CHECK(ws && ws_bytes >= novic_preference_loss_ws(n, T), "novic_preference_loss: the workspace is smaller than novic_preference_loss_ws says");
	NOVIC_APART("novic_preference_loss",
	            NOVIC_SPANS(dlogits_span(g, type), vector_span(stats, 12), vector_span(margin, 4LL * n), token_span(g, logp, ldo), vector_span(ws, novic_preference_loss_ws(n, T))),
	            NOVIC_SPANS(target_span(g), pad_span(g), token_span(g, ref, ldref), vector_span(weight, 4LL * n)), NOVIC_SPANS(logits_span(g, type)))
	const uint64_t R = 2ull * n * T;
	char* w = (char*)ws;
	double* diff = (double*)w; w += up16(8 * R);
	double* each = (double*)w; w += up16(16ull * n);
	float2* norm = (float2*)w; w += up16(8 * R);
	float* coef = (float*)w; w += up16(8ull * n);
	float* scale = (float*)w;
	LogpOut o = {};
	o.logp = logp; o.ldo = ldo; o.ref = ref; o.ldref = ldref; o.diff = diff; o.norm = dlogits ? norm : nullptr;
	NOVIC_ROW_TYPES(type, V, launch_logp, g, o, stream)
	Pref q = {diff, weight, n, T, kind, beta, smoothing, grad_scale, margin, coef, each, scale, stats};
	const int lanes = lanes_for(T);
	pref_pair_kernel<<<dim3((unsigned)(((long long)n * lanes + 255) / 256)), dim3(256), 0, stream>>>(q, lanes);
	pref_finish_kernel<<<dim3(1), dim3(1024), 0, stream>>>(q);
	if (dlogits) {
		GradIn in = {};
		in.norm = norm; in.grad = coef; in.lda = 1; in.ldt = 0; in.scale = scale;
		NOVIC_ROW_TYPES(type, V, launch_grad, g, in, stream)
	}
	NOVIC_LAUNCH_CHECK();
	return 0;
}

// workspace: len [A], part [2][64], each [3][A T]
extern "C" uint64_t novic_policy_loss_ws(int A, int T) {
	if (A <= 0 || T <= 0) return 0;
	return up16(4ull * A) + up16(8 * COUNT_PARTS) + 12ull * A * T;
}
extern "C" int novic_policy_loss(const void* logits, int type, int64_t ldl, const void* target, int tok_bytes, int64_t ldt, const uint8_t* pad, int64_t ldp, int A, int T, int V,
                                 const float* old_logp, int64_t ldold, const float* adv, int64_t adv_lda, int64_t adv_ldt, const float* ref, int64_t ldref, float clip_lo, float clip_hi,
                                 float kl_coef, int per_sequence, float grad_scale, float* logp, int64_t ldo, void* dlogits, int64_t ldd, float* stats, void* ws, uint64_t ws_bytes,
                                 hipStream_t stream) {
	NOVIC_CHECK(A >= 1 && T >= 1, "novic_policy_loss: at least one sequence and one position");
	Rows g = {logits, ldl, dlogits, ldd, target, pad, ldt, ldp, tok_bytes, A, T, V};
	const char* bad = rows_bad(g, type);
	NOVIC_CHECK(!bad, bad);
	NOVIC_CHECK(old_logp && adv && stats && (A <= 1 || (ldold >= T && (!ref || ldref >= T) && (!logp || ldo >= T))), "novic_policy_loss: old, ref, logp [A][ld >= T], stats [4]");
	NOVIC_CHECK(clip_lo >= 0.f && clip_lo <= 1.f && clip_hi >= 0.f && kl_coef >= 0.f, "novic_policy_loss: 0 <= clip_lo <= 1, clip_hi >= 0, kl_coef >= 0");
	NOVIC_CHECK(ws && ws_bytes >= novic_policy_loss_ws(A, T), "novic_policy_loss: the workspace is smaller than novic_policy_loss_ws says");
	NOVIC_CHECK(adv_ldt == 0 || adv_ldt == 1, "novic_policy_loss: adv has unit stride along the positions, or one value a sequence");
	NOVIC_APART("novic_policy_loss", NOVIC_SPANS(dlogits_span(g, type), vector_span(stats, 16), token_span(g, logp, ldo), vector_span(ws, novic_policy_loss_ws(A, T))),
	            NOVIC_SPANS(target_span(g), pad_span(g), token_span(g, old_logp, ldold), token_span(g, ref, ldref), {adv, A, adv_ldt ? 4LL * T : 4, 4 * adv_lda}),
	            NOVIC_SPANS(logits_span(g, type)))
	Policy p = {};
	p.old = old_logp; p.adv = adv; p.ref = ref;
	p.ldold = ldold; p.ldref = ldref; p.lda = adv_lda; p.ldt = adv_ldt;
	p.lo = clip_lo; p.hi = clip_hi; p.kl_coef = kl_coef; p.grad_scale = grad_scale;
	p.per_seq = per_sequence;
	p.logp = logp; p.ldo = ldo;
	char* w = (char*)ws;
	p.len = (int*)w; w += up16(4ull * A);
	p.part = (int*)w; w += up16(8 * COUNT_PARTS);
	p.each = (float*)w;
	p.parts = count_parts(A, T);
	p.stats = stats;
	policy_count_kernel<<<dim3(p.parts), dim3(256), 0, stream>>>(g, p, lanes_for(T));
	NOVIC_ROW_TYPES(type, V, launch_policy, g, p, stream)
	policy_finish_kernel<<<dim3(1), dim3(1024), 0, stream>>>(g, p);
	NOVIC_LAUNCH_CHECK();
	return 0;
}
