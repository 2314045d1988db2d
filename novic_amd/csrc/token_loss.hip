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
// Exponentials, sums over the vocabulary and the logarithm of such a sum are fp32; what they give is added to the maximum, and up over a sequence, in fp64 (a handful of operations
// a ROW): the losses take differences of sums that nearly cancel.  A log-probability is off by some 1e-7: at 7 000 to 50 000 columns of scale 2 by -5e-8 on average (log2 e rounds
// down, which makes the exponentials below the maximum a little large), 5e-8 to 7e-8 rms about that.  The average adds up over a sequence, to 1.7e-5 in 333 tokens, where the rounding
// of their fp32 reference values (up to 2^-21 each at -10) adds 5e-6.  A second part of log2 e does not mend it: most of it is lost in the rounding of the fp32 exponent.
// MI355X: gradient of log-probabilities over [4928 x 49408] fp16 137 us (733 MB, 5.4 TB/s); preference step of 4096 pairs of [7 x 6912] bf16 250 us (1249 MB, 5.0 TB/s), policy step
// of as many rows 219 us (5.7 TB/s); each back to back, some 20 us more for a call that finds the GPU idle.
#include "novic_hip.h"
#include "rowvec.hpp"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
// A row's sums are seen from M = fl(m log2 e), m its maximum: an exponential is one fma and one v_exp_f32, exp2(x LOG2E - M), and M's rounding takes part in nothing but the choice
// of the point, m' = M / LOG2E, from which x - m' is measured (in fp64, once a row).  Beyond FAR (a row that is masked with -1e30 or its type's lowest value throughout) that rounding
// would be 64 and more, and the product need not be a number.  Two numbers there are equal or differ by 128 at least, so that powers of two tell them apart as well as
// exponentials do: m is the point itself.
constexpr float FAR = 1.4e9f;
struct Point {
	float M, L;
};
__device__ __forceinline__ Point point(float m) {
	const bool far = fabsf(m) > FAR;
	return {far ? m : m * LOG2E, far ? 1.f : LOG2E};
}
__device__ __forceinline__ float expo(float x, Point p) { return __builtin_amdgcn_exp2f(fmaf(x, p.L, -p.M)); }
__device__ __forceinline__ double from_point(float m) {  // m'
	return fabsf(m) > FAR ? (double)m : (double)(m * LOG2E) * (1.0 / (double)LOG2E);
}
// what a sum seen from the point of `from` is multiplied by to be seen from that of `to`
__device__ __forceinline__ float shift(float from, float to) {
	const Point a = point(from), b = point(to);
	return a.L == b.L ? __builtin_amdgcn_exp2f(a.M - b.M) : 0.f;
}

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

__device__ __forceinline__ int counted_target(const Rows& g, int a, int t) {  // -1: the position does not count (mask and target are requested together)
	const bool padded = g.pad && g.pad[a * g.ldp + t];
	const long long v = g.tok_bytes == 8 ? ((const long long*)g.target)[a * g.ldt + t] : (long long)((const int*)g.target)[a * g.ldt + t];
	return padded || v < 0 || v >= g.V ? -1 : (int)v;
}

// Workgroup -> row.  A grid's extent in threads is 32 bits, so rows beyond 2^20 go to its second dimension.
__device__ __forceinline__ int row_index(const Rows& g) {
	const long long r = (long long)blockIdx.y * gridDim.x + blockIdx.x;
	return r < (long long)g.A * g.T ? (int)r : -1;
}

// log(s) of a sum to 3e-8 ABSOLUTE, however large, without the cost of a double-precision logarithm: s = 2^k f, f in [0.7, 1.42), |logf(f)| < 0.36; the sum itself is off by more
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
		const Point at_m = point(m);
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
				x[c][i] = expo(x[c][i], at_m);
				if ((c + 1) * THREADS * CH > V && at(c, V) + i < own(c)) x[c][i] = 0.f;
				t += x[c][i];
			}
		}
		s = block_sum<THREADS>(t, red + THREADS / 64);
	}
	// dlogits = g ([v = target] - x / s); the target's element is stored once more by the lane that owns it, which costs less than a comparison an element
	__device__ __forceinline__ void grad(T* row, int V, int target, float et, float g) {
		const float k = -g / s;
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			if (own(c) >= V) continue;
			float o[CH];
#pragma unroll
			for (int i = 0; i < CH; ++i) o[i] = k * x[c][i];
			store_own<true>(row, at(c, V), own(c), o);
		}
		if ((target / CH) % THREADS == (int)threadIdx.x) row[target] = (T)(k * et + g);
	}
};

// A row in passing, by a team of LANES lanes: UNROLL vectors a lane are requested at once.
template <typename T, int CH, int LANES, int UNROLL = 4>
struct RowStream {
	// (vectors that all lanes have whole are addressed from a scalar base and the one offset of the lane)
	__device__ __forceinline__ static void load(RawVec<T, CH> (&raw)[UNROLL], const T* row, int e, int V, int lane) {
		if (e + UNROLL * LANES * CH <= V) {
#pragma unroll
			for (int u = 0; u < UNROLL; ++u) raw[u] = load_vec<T, CH>(elem(row + (e + u * LANES * CH), lane * CH));
		} else {
#pragma unroll
			for (int u = 0; u < UNROLL; ++u) raw[u] = load_vec<T, CH>(elem(row, min(e + (u * LANES + lane) * CH, V - CH)));
		}
	}
	// maximum and sum over this lane's part; the next vectors are requested before the present ones are added
	__device__ __forceinline__ static void sum(const T* row, int V, int lane, float& tm, float& ts) {
		tm = -INFINITY;
		ts = 0.f;
		RawVec<T, CH> raw[UNROLL], next[UNROLL];
		load(raw, row, 0, V, lane);
		for (int e = 0; e < V; e += UNROLL * LANES * CH) {
			if (e + UNROLL * LANES * CH < V) load(next, row, e + UNROLL * LANES * CH, V, lane);
			float top = -INFINITY;
#pragma unroll
			for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
				for (int i = 0; i < CH; ++i) top = fmaxf(top, raw[u].get(i));
				forget(raw[u]);  // (else its elements stay unpacked from one use to the next, at twice the registers)
			}
			const float m = fmaxf(tm, top), base = m == -INFINITY ? 0.f : m;  // (nothing but -inf yet: their exponentials are zeros)
			const Point at_m = point(base);
			ts *= shift(tm, base);
			if (e + UNROLL * LANES * CH <= V) {
#pragma unroll
				for (int u = 0; u < UNROLL; ++u)
#pragma unroll
					for (int i = 0; i < CH; ++i) ts += expo(raw[u].get(i), at_m);
			} else {
#pragma unroll
				for (int u = 0; u < UNROLL; ++u) {
					const int e0 = e + (u * LANES + lane) * CH, es = min(e0, V - CH);
#pragma unroll
					for (int i = 0; i < CH; ++i) ts += es + i >= e0 ? expo(raw[u].get(i), at_m) : 0.f;
				}
			}
			tm = m;
#pragma unroll
			for (int u = 0; u < UNROLL; ++u) raw[u] = next[u];
		}
	}
	// a lane's sum seen from the row's point
	__device__ __forceinline__ static float scaled(float tm, float ts, float m) { return ts * shift(tm, m == -INFINITY ? 0.f : m); }
	// out = k exp(x - m), and coef more at the target (whose logit is xt); out may be row
	__device__ __forceinline__ static void grad(const T* row, T* out, int V, int lane, int target, float xt, float m, float k, float coef) {
		const Point at_m = point(m);
		RawVec<T, CH> raw[UNROLL], next[UNROLL];
		load(raw, row, 0, V, lane);
		// xt may come through the scalar cache, whose loads are not ordered with vector stores: it has to be here before the first of them, where out is row
		asm volatile("" : "+v"(xt));
		for (int e = 0; e < V; e += UNROLL * LANES * CH) {
			if (e + UNROLL * LANES * CH < V) load(next, row, e + UNROLL * LANES * CH, V, lane);  // (before this piece's stores, also where out is row: no vector is in both)
#pragma unroll
			for (int u = 0; u < UNROLL; ++u) {
				float o[CH];
#pragma unroll
				for (int i = 0; i < CH; ++i) o[i] = k * expo(raw[u].get(i), at_m);
				if (e + UNROLL * LANES * CH <= V) {
					store_vec<true>(elem(out + (e + u * LANES * CH), lane * CH), o);
				} else {
					const int e0 = e + (u * LANES + lane) * CH;
					if (e0 < V) store_own<true>(out, min(e0, V - CH), e0, o);
				}
			}
#pragma unroll
			for (int u = 0; u < UNROLL; ++u) raw[u] = next[u];
		}
		if ((target / CH) % LANES == lane) out[target] = (T)(k * expo(xt, at_m) + coef);
	}
	__device__ __forceinline__ static void zero(T* row, int V, int lane) {
		float o[CH];
#pragma unroll
		for (int i = 0; i < CH; ++i) o[i] = 0.f;
		for (int e0 = lane * CH; e0 < V; e0 += LANES * CH) store_own<true>(row, min(e0, V - CH), e0, o);
	}
};

// A row in the registers of a team of LANES lanes (16 or 64), as it lies in memory.  Vector c of all lanes together is the STEP elements from c STEP on; where those would leave the row it is the row's
// last STEP elements, of which the first cut(c) belong to vectors before it: a scalar base and one offset a lane address everything, and no load is conditional (a conditional
// one in a loop costs a second copy of the registers).  NC = 1: a row of at most STEP elements, each lane's vector moved back by itself.
template <typename T, int CH, int LANES, int NC>
struct TeamRow {
	static constexpr int STEP = LANES * CH;
	RawVec<T, CH> raw[NC];
	__device__ __forceinline__ static int base(int c, int V) { return NC == 1 ? 0 : min(c * STEP, V - STEP); }
	__device__ __forceinline__ static int at(int V, int lane) { return NC == 1 ? min(lane * CH, V - CH) : lane * CH; }
	__device__ __forceinline__ static int cut(int c, int V, int lane) { return NC == 1 ? lane * CH : c * STEP - base(c, V); }  // first element of at() .. that counts
	__device__ __forceinline__ static bool whole(int c, int V) { return (c + 1) * STEP <= V; }
	__device__ __forceinline__ static bool any(int c, int V) { return c * STEP < V; }
	// What a row's end needs (NC CH masks of lanes, NC bases) is the same in every row: formed for all rows at once it would fill the scalar registers many times over.  So each use
	// forms its own, and only the vector at the end has any.
	__device__ __forceinline__ static void here(int& V, int& lane) {
		if constexpr (NC > 1) asm volatile("" : "+s"(V), "+v"(lane));
	}
	__device__ __forceinline__ void load(const T* row, int V, int lane) {
		here(V, lane);
#pragma unroll
		for (int c = 0; c < NC; ++c) raw[c] = load_vec<T, CH>(elem(row + base(c, V), at(V, lane)));
	}
	// The maximum of 16-bit elements two at a time, as integers: a number that is not negative compares as its bits do, and above every negative one.  Only a row whose maximum
	// comes out negative is looked over again, element by element (there the bits of the lowest number win).
	__device__ __forceinline__ float top() {
		float t = -INFINITY;
		if constexpr (sizeof(T) == 2 && CH > 1) {
			typedef short pair __attribute__((ext_vector_type(2)));
			pair best = {(short)0x8000, (short)0x8000};
#pragma unroll
			for (int c = 0; c < NC; ++c)
#pragma unroll
				for (int i = 0; i < CH / 2; ++i) {
					pair p;
					__builtin_memcpy(&p, &raw[c].w[i], 4);
					best = __builtin_elementwise_max(best, p);
				}
			RawVec<T, 2> r;
			__builtin_memcpy(&r, &best, 4);
			t = team_max<LANES>(fmaxf(r.get(0), r.get(1)));
			if (t > 0.f) return t;
			t = -INFINITY;
		}
#pragma unroll
		for (int c = 0; c < NC; ++c) {
#pragma unroll
			for (int i = 0; i < CH; ++i) t = fmaxf(t, raw[c].get(i));
			forget(raw[c]);
		}
		return team_max<LANES>(t);
	}
	// (where the team is a wave the point goes to scalar registers)
	__device__ __forceinline__ static Point at_max(float m) { return point(LANES == 64 ? __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(m))) : m); }
	__device__ __forceinline__ void sum(int V, int lane, float& m, float& s) {
		m = top();
		const Point at_m = at_max(m == -INFINITY ? 0.f : m);  // (nothing but -inf: a sum of zeros, whose logarithm is -inf)
		here(V, lane);
		float t = 0.f;
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			forget(raw[c]);  // (else its elements stay unpacked from one use to the next, at twice the registers)
			if (whole(c, V)) {
#pragma unroll
				for (int i = 0; i < CH; ++i) t += expo(raw[c].get(i), at_m);
			} else if (any(c, V)) {
#pragma unroll
				for (int i = 0; i < CH; ++i) t += at(V, lane) + i >= cut(c, V, lane) ? expo(raw[c].get(i), at_m) : 0.f;
			}
		}
		s = team_sum<LANES>(t);
	}
	__device__ __forceinline__ void grad(T* out, int V, int lane, int target, float xt, float m, float k, float coef) {
		const Point at_m = at_max(m);
		asm volatile("" : "+v"(xt));  // (as in RowStream)
		here(V, lane);
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			if (!any(c, V)) continue;
			forget(raw[c]);
			float o[CH];
#pragma unroll
			for (int i = 0; i < CH; ++i) o[i] = k * expo(raw[c].get(i), at_m);
			if (whole(c, V)) {
				store_vec<true>(elem(out + base(c, V), at(V, lane)), o);
			} else if (at(V, lane) >= cut(c, V, lane)) {
				store_vec<true>(elem(out + base(c, V), at(V, lane)), o);
			} else {
#pragma unroll
				for (int i = 1; i < CH; ++i)
					if (at(V, lane) + i >= cut(c, V, lane) && cut(c, V, lane) < V) *elem(out + base(c, V), at(V, lane) + i) = (T)o[i];
			}
		}
		if (owner(target, V) == lane) out[target] = (T)(k * expo(xt, at_m) + coef);
	}
	// the lane that stores element v (after which it may store it once more)
	__device__ __forceinline__ static int owner(int v, int V) {
		if (NC == 1) return v / CH;
		return v / STEP * STEP <= V - STEP ? v % STEP / CH : (v - (V - STEP)) / CH;
	}
};

// Rows by team: the teams of a launch walk over the rows.  A row's mask and target are requested while the row before it is worked on, and looked at when its turn comes.
template <int LANES>
struct Walk {
	int r, step, a, t;
	bool padded;
	long long id;
	// (where a team is a wave, what is the same for it goes to scalar registers)
	__device__ __forceinline__ static int same(int v) { return LANES == 64 ? __builtin_amdgcn_readfirstlane(v) : v; }
	__device__ __forceinline__ Walk(const Rows& g) : r(same(blockIdx.x * (256 / LANES) + threadIdx.x / LANES)), step(gridDim.x * (256 / LANES)) { ask(g); }
	__device__ __forceinline__ void ask(const Rows& g) {
		a = r / g.T;
		t = r - a * g.T;
		padded = true;
		id = -1;
		if (done(g)) return;
		padded = g.pad && g.pad[a * g.ldp + t];
		id = g.tok_bytes == 8 ? ((const long long*)g.target)[a * g.ldt + t] : (long long)((const int*)g.target)[a * g.ldt + t];
	}
	__device__ __forceinline__ int target(const Rows& g) const { return same(padded || id < 0 || id >= g.V ? -1 : (int)id); }
	__device__ __forceinline__ bool done(const Rows& g) const { return r >= g.A * g.T; }
	__device__ __forceinline__ Walk next(const Rows& g) const {
		Walk n = *this;
		n.r = r > 0x7fffffff - step ? 0x7fffffff : r + step;
		n.ask(g);
		return n;
	}
};

// ---- log-probabilities -------------------------------------------------------------------------------------------------------------------------------------------
struct LogpOut {
	float* logp;       // [A][T] or null
	float* lse;        // [A T] or null: the row's log-sum-exp
	const float* ref;  // [A][T] or null
	double* diff;      // [A T] or null: lp - ref, 0 where the row does not count
	float2* norm;      // [A T] or null: (m, 1 / s)
	long long ldo, ldref;
};
__device__ __forceinline__ float reference(const LogpOut& o, int a, int t) { return o.diff ? o.ref[a * o.ldref + t] : 0.f; }
__device__ __forceinline__ void put_logp(const LogpOut& o, int r, int a, int t, bool counts, double lp, float m, float s, float ref = 0.f) {
	if (o.logp) o.logp[a * o.ldo + t] = counts ? (float)lp : 0.f;
	if (o.lse) o.lse[r] = counts ? (float)(from_point(m) + log_wide(s)) : 0.f;
	if (o.diff) o.diff[r] = counts ? lp - (double)ref : 0.0;
	if (o.norm) o.norm[r] = counts ? make_float2(m, 1.f / s) : make_float2(0.f, 0.f);
}

template <typename T, int CH, int THREADS, int UNROLL = 4>
__device__ __forceinline__ void block_row_sum(const T* row, int V, float* red, float& m, float& s) {
	typedef RowStream<T, CH, THREADS, UNROLL> Stream;
	float tm, ts;
	Stream::sum(row, V, threadIdx.x, tm, ts);
	m = block_max<THREADS>(tm, red);
	s = block_sum<THREADS>(Stream::scaled(tm, ts, m), red + THREADS / 64);
}
__device__ __forceinline__ double row_logp(float xt, float m, float s) { return ((double)xt - from_point(m)) - log_wide(s); }
template <typename T, int CH, int THREADS>
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
	const float xt = (float)row[target], ref = reference(o, a, t);
	float m, s;
	block_row_sum<T, CH, THREADS>(row, g.V, red, m, s);
	if (threadIdx.x == 0) put_logp(o, r, a, t, true, row_logp(xt, m, s), m, s, ref);
}

template <typename T, int CH, int LANES, int NC>
__global__ __launch_bounds__(256) void logp_team_kernel(const Rows g, const LogpOut o) {
	const int lane = threadIdx.x % LANES;
	TeamRow<T, CH, LANES, NC> tile;
	Walk<LANES> now(g);
	while (!now.done(g)) {
		const int target = now.target(g);
		float xt = 0.f, ref = 0.f;
		if (target >= 0) {
			const T* row = (const T*)g.logits + (long long)now.r * g.ldl;
			tile.load(row, g.V, lane);
			xt = (float)row[target];
			ref = reference(o, now.a, now.t);
		}
		const Walk<LANES> next = now.next(g);
		float m = 0.f, s = 1.f;
		if (target >= 0) tile.sum(g.V, lane, m, s);
		if (lane == 0) put_logp(o, now.r, now.a, now.t, target >= 0, target >= 0 ? row_logp(xt, m, s) : 0.0, m, s, ref);
		now = next;
	}
}

// ---- gradient of log-probabilities: dlogits = coef (1[v = target] - exp(x - m) / s) ----------------------------------------------------------------------------------
struct GradIn {
	const float* lse;     // [A T], or null:
	const float2* norm;   // [A T] (m, 1 / s)
	const float* grad;    // element (a, t) at grad[a * lda + t * ldt]
	long long lda, ldt;
	const float* scale;   // device scalar or null
};
// An lse beyond COARSE has lost what its rounding (2^-16 and more) takes from every probability, at 1e9 all of log V: there the row's sum is formed again, at a second read, and used if
// lse is its rounding (one that is not, such as that of a vocabulary of which these are some columns, stands as it is).  By one vector at a time: such rows are rare, and more would
// take registers from the others.
constexpr float COARSE = 256.f;
// (lse and the point from which s is seen are each off by 2^-24 of themselves, their difference rounds once more)
__device__ __forceinline__ bool rounds_to(float m, float s, float lse) { return fabsf((m - lse) + logf(s)) <= fabsf(lse) * 0x1p-22f; }
// dlogits = k exp(x - m) + (coef at the target); sums(m, s): the row's maximum and sum
template <typename Sums>
__device__ __forceinline__ void grad_terms(const GradIn& in, int r, int a, int t, float& m, float& k, float& coef, Sums sums) {
	coef = in.grad[a * in.lda + t * in.ldt];
	if (in.scale) coef *= *in.scale;
	k = -coef;
	if (in.norm) {
		const float2 n = in.norm[r];
		m = n.x;
		k *= n.y;
		return;
	}
	const float lse = in.lse[r];
	if (fabsf(lse) > COARSE) {
		float s;
		sums(m, s);
		if (rounds_to(m, s, lse)) {
			k /= s;
			return;
		}
	}
	m = lse;
	const Point at_m = point(m);
	k *= __builtin_amdgcn_exp2f(-fmaf(m, at_m.L, -at_m.M));  // (what the point's rounding took: s is what lse says, seen from M)
}
template <typename T, int CH, int THREADS>
__global__ __launch_bounds__(THREADS) void logp_grad_kernel(const Rows g, const GradIn in) {
	__shared__ float red[2 * THREADS / 64];
	const int r = row_index(g);
	if (r < 0) return;
	const int a = r / g.T, t = r - a * g.T;
	const int target = counted_target(g, a, t);
	T* out = (T*)g.dlogits + (long long)r * g.ldd;
	if (target < 0) {
		RowStream<T, CH, THREADS>::zero(out, g.V, threadIdx.x);
		return;
	}
	const T* row = (const T*)g.logits + (long long)r * g.ldl;
	float m, k, coef;
	grad_terms(in, r, a, t, m, k, coef, [&](float& top, float& s) { block_row_sum<T, CH, THREADS, 1>(row, g.V, red, top, s); });
	const float xt = (float)row[target];  // (used by the lane that owns the target alone, which loads it before it writes there: out may be row)
	RowStream<T, CH, THREADS>::grad(row, out, g.V, threadIdx.x, target, xt, m, k, coef);
}

template <typename T, int CH, int LANES>
__global__ __launch_bounds__(256) void logp_grad_team_kernel(const Rows g, const GradIn in) {
	typedef RowStream<T, CH, LANES> Stream;
	const int lane = threadIdx.x % LANES;
	Walk<LANES> now(g);
	while (!now.done(g)) {
		const int target = now.target(g);
		T* out = (T*)g.dlogits + (long long)now.r * g.ldd;
		const Walk<LANES> next = now.next(g);
		if (target < 0) {
			Stream::zero(out, g.V, lane);
		} else {
			const T* row = (const T*)g.logits + (long long)now.r * g.ldl;
			float m, k, coef;
			grad_terms(in, now.r, now.a, now.t, m, k, coef, [&](float& top, float& s) {
				typedef RowStream<T, CH, LANES, 1> Slow;
				float tm, ts;
				Slow::sum(row, g.V, lane, tm, ts);
				top = team_max<LANES>(tm);
				s = team_sum<LANES>(Slow::scaled(tm, ts, top));
			});
			Stream::grad(row, out, g.V, lane, target, (float)row[target], m, k, coef);
		}
		now = next;
	}
}

// ---- preference loss ---------------------------------------------------------------------------------------------------------------------------------------------
struct Pref {
	const double* diff;   // [2 n][T]
	const float* weight;  // [n] or null
	int n, T, kind;
	double beta, smoothing, grad_scale;
	float* margin;        // [n] or null
	float* coef;          // [2 n]: gradient of sum_i w_i l_i to a sequence's u
	double* each;         // [2][n]: w l, w z
	double* total;        // device scalar: sum(w), or null
	float* scale;         // device scalar: grad_scale / sum(w)
	float* stats;         // [3]: loss, mean margin, sum(w)
};
__device__ __forceinline__ double pref_margin(const Pref& g, double up, double un) { return g.beta * (up - un); }
__device__ __forceinline__ float pref_weight(const Pref& g, int i) { return g.weight ? g.weight[i] : 1.f; }
// gradient of sum_i w_i l_i to u of pair i's preferred sequence (the other's is its negative).  A sigmoid's small side is formed by itself, without a difference, in fp32; the square
// form and the products are fp64: 1 / beta^2 may leave fp32 where the slope, which takes beta once more, does not.
__device__ __forceinline__ float pref_slope(const Pref& g, int i, double z) {
	double du;
	if (g.kind == NOVIC_PREF_SQUARE) {
		du = 2.0 * (z - 0.5) / g.beta;
	} else {
		float dz;
		if (g.kind == NOVIC_PREF_SIGMOID) {
			const float e = expf(-fabsf((float)z)), small = e / (1.f + e), large = 1.f / (1.f + e);
			const float at = z < 0.0 ? small : large, rest = z < 0.0 ? large : small;  // sigmoid(z), sigmoid(-z)
			dz = (float)g.smoothing * at - (1.f - (float)g.smoothing) * rest;
		} else {
			dz = z < 1.0 ? -1.f : (z >= 1.0 ? 0.f : (float)z);  // (a NaN stays one)
		}
		du = (double)dz * g.beta;
	}
	return (float)((double)pref_weight(g, i) * du);
}
__device__ __forceinline__ void pref_terms(const Pref& g, int i, double z) {
	double l;
	if (g.kind == NOVIC_PREF_SIGMOID) {
		const double soft = log1p(exp(-fabs(z)));  // -log sigmoid(z) = soft + max(-z, 0)
		l = (1.0 - g.smoothing) * (soft + fmax(-z, 0.0));
		if (g.smoothing != 0.0) l += g.smoothing * (soft + fmax(z, 0.0));  // (a margin of +inf, whose rejected label has an excluded token, costs nothing without it)
	} else if (g.kind == NOVIC_PREF_HINGE) {
		l = z < 1.0 ? 1.0 - z : (z >= 1.0 ? 0.0 : z);
	} else {
		const double u = (z - 0.5) / g.beta;
		l = u * u;
	}
	const double w = (double)pref_weight(g, i);
	if (g.margin) g.margin[i] = (float)z;
	g.each[i] = w * l;
	g.each[g.n + i] = w * z;
}
// sum of one sequence's T values by `lanes` consecutive lanes (a power of two up to 64), in a fixed order
__device__ __forceinline__ double seq_sum(const double* v, int T, int lane, int lanes) {
	double u = 0.0;
	for (int t0 = lane; t0 < T; t0 += 8 * lanes) {  // eight values a lane requested at once
		double part[8];
#pragma unroll
		for (int k = 0; k < 8; ++k) part[k] = v[min(t0 + k * lanes, T - 1)];
#pragma unroll
		for (int k = 0; k < 8; ++k) u += t0 + k * lanes < T ? part[k] : 0.0;
	}
	for (int o = lanes / 2; o > 0; o >>= 1) u += __shfl_xor(u, o, 64);
	return u;
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
// what a mean over the weights w sums to: the scale of the gradients and, from the sums of w l and w z, the three numbers of a call
__device__ __forceinline__ float pref_scale(const Pref& g, double w) { return w != 0.0 ? (float)(g.grad_scale / w) : 0.f; }  // (no weight at all: no loss and no gradient)
__device__ __forceinline__ void pref_stats(const Pref& g, double l, double z, double w) {
	g.stats[0] = w != 0.0 ? (float)(l / w) : 0.f;
	g.stats[1] = w != 0.0 ? (float)(z / w) : 0.f;
	g.stats[2] = (float)w;
}
// the pairs' terms and their coefficients by many workgroups; pref_finish_kernel adds the terms
__global__ __launch_bounds__(256) void pref_each_kernel(const Pref g, int lanes) {
	const int lane = threadIdx.x % lanes, i = (int)(((long long)blockIdx.x * 256 + threadIdx.x) / lanes);
	if (i >= g.n) return;
	const double up = seq_sum(g.diff + (long long)i * g.T, g.T, lane, lanes), un = seq_sum(g.diff + ((long long)g.n + i) * g.T, g.T, lane, lanes);
	if (lane != 0) return;
	const double m = pref_margin(g, up, un);
	const float c = pref_slope(g, i, m);
	pref_terms(g, i, m);
	g.coef[i] = c;
	g.coef[g.n + i] = -c;
}
// all pairs, by one workgroup: the sums over the sequences, the pairs' terms and their coefficients, the three numbers
__global__ __launch_bounds__(1024) void pref_all_kernel(const Pref g, int lanes) {
	__shared__ double red[48];
	const int lane = threadIdx.x % lanes, teams = 1024 / lanes;
	double l = 0.0, z = 0.0, w = 0.0;
	for (int i = threadIdx.x / lanes; i < g.n; i += teams) {
		const double up = seq_sum(g.diff + (long long)i * g.T, g.T, lane, lanes), un = seq_sum(g.diff + ((long long)g.n + i) * g.T, g.T, lane, lanes);
		if (lane == 0) {
			const double m = pref_margin(g, up, un);
			const float c = pref_slope(g, i, m);
			pref_terms(g, i, m);
			g.coef[i] = c;
			g.coef[g.n + i] = -c;
			l += g.each[i];
			z += g.each[g.n + i];
			w += (double)pref_weight(g, i);
		}
	}
	sum3_1024(l, z, w, red);
	if (threadIdx.x == 0) {
		pref_stats(g, l, z, w);
		*g.scale = pref_scale(g, w);
	}
}
// sum of the weights, for the form that makes gradients pair by pair
__global__ __launch_bounds__(1024) void pref_weight_kernel(const Pref g) {
	__shared__ double red[48];
	double w = 0.0, a = 0.0, b = 0.0;
	for (int i = threadIdx.x; i < g.n; i += 1024) w += (double)g.weight[i];
	sum3_1024(w, a, b, red);
	if (threadIdx.x == 0) *g.total = w;
}
__global__ __launch_bounds__(1024) void pref_finish_kernel(const Pref g) {
	__shared__ double red[48];
	double l = 0.0, z = 0.0, w = 0.0;
	for (int i0 = threadIdx.x; i0 < g.n; i0 += 4 * 1024) {  // four pairs a thread requested at once
		double a[4], b[4];
		float c[4];
#pragma unroll
		for (int k = 0; k < 4; ++k) {
			const int i = min(i0 + k * 1024, g.n - 1);
			a[k] = g.each[i];
			b[k] = g.each[g.n + i];
			c[k] = pref_weight(g, i);
		}
#pragma unroll
		for (int k = 0; k < 4; ++k) {
			if (i0 + k * 1024 >= g.n) continue;
			l += a[k];
			z += b[k];
			w += (double)c[k];
		}
	}
	sum3_1024(l, z, w, red);
	if (threadIdx.x == 0) {
		pref_stats(g, l, z, w);
		*g.scale = pref_scale(g, w);
	}
}

// A pair by one workgroup, loss and gradient.  The pair's rows (at most 64) are lanes' business first: each wave asks for all targets and reference values and knows the rows that
// count from a ballot.  Those are dealt to the waves in turn; the row that a wave sums last stays in its registers up to its gradient, any others are read again (a pair's
// time later: out of L2 or the memory-side cache).  Sixteen vectors a lane are what 128 registers hold beside the rest of the kernel.  Bound by the rows in flight: between a pair's
// reading and its writing stands a barrier, and two workgroups a unit are what covers it.  4096 pairs of 7 + 7 rows of 6912 bf16: 249 us with eight waves, with four 272.
// Second rows kept in LDS instead of read again: 1 % less.
constexpr int PAIR_ROWS = 64, PAIR_VECTORS = 16, PAIR_WEIGHTS = 4096;
template <typename T, int CH, int NC, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 4) void pref_pair_kernel(const Rows g, const LogpOut o, const Pref q) {
	__shared__ double part[3][WAVES];
	const int i = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, rows = 2 * q.T;
	const int my_half = lane >= q.T, my_a = my_half ? q.n + i : i, my_t = lane - my_half * q.T;  // lane k stands for row k: the preferred sequence's, then the other's
	int my_target = -1;
	float my_ref = 0.f;
	if (lane < rows) {
		my_target = counted_target(g, my_a, my_t);
		my_ref = o.ref[my_a * o.ldref + my_t];
	}
	double total = 0.0;  // of the weights: few enough are added up by every workgroup (q.total is null), which saves a launch in front of this one
	if (q.weight && !q.total) {
		float w[PAIR_WEIGHTS / (WAVES * 64)];
#pragma unroll
		for (int k = 0; k < PAIR_WEIGHTS / (WAVES * 64); ++k) w[k] = q.weight[min(k * WAVES * 64 + (int)threadIdx.x, q.n - 1)];
#pragma unroll
		for (int k = 0; k < PAIR_WEIGHTS / (WAVES * 64); ++k) total += k * WAVES * 64 + (int)threadIdx.x < q.n ? (double)w[k] : 0.0;
#pragma unroll
		for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
	}
	const unsigned long long counted = __ballot(my_target >= 0), others = __ballot(lane < rows && my_target < 0);
	const int have = __popcll(counted), none = __popcll(others);
	auto nth = [&](unsigned long long set, int l) {  // the l-th member of a set of lanes
		return __ffsll((unsigned long long)__ballot(((set >> lane) & 1) && __popcll(set & ((1ull << lane) - 1)) == l)) - 1;
	};
	auto row_of = [&](int k) { return (k >= q.T ? q.n + i : i) * q.T + (k >= q.T ? k - q.T : k); };
	auto of_lane = [&](int v, int k) { return __builtin_amdgcn_readlane(v, k); };
	double u[2] = {0.0, 0.0};
	auto counted_row = [&](int k, int r, float xt, float m, float s) {  // lane 0: the row's log-probability, added to its sequence
		const double lp = row_logp(xt, m, s), d = lp - (double)__int_as_float(of_lane(__float_as_int(my_ref), k));
		u[0] += k >= q.T ? 0.0 : d;
		u[1] += k >= q.T ? d : 0.0;
		if (lane == 0) put_logp(o, r, k >= q.T ? q.n + i : i, k >= q.T ? k - q.T : k, true, lp, m, s);
	};
	TeamRow<T, CH, 64, NC> tile;
	float m = 0.f, s = 1.f, xt = 0.f;
	int k = 0, r = 0, target = 0;
	for (int l = wave + (have - 1 - wave) / WAVES * WAVES; wave < have && l >= 0; l -= WAVES) {
		k = nth(counted, l), r = row_of(k), target = of_lane(my_target, k);
		const T* row = (const T*)g.logits + (long long)r * g.ldl;
		tile.load(row, g.V, lane);
		xt = (float)row[target];
		tile.sum(g.V, lane, m, s);
		counted_row(k, r, xt, m, s);
	}
	if (lane == 0) {
		part[0][wave] = u[0];
		part[1][wave] = u[1];
		part[2][wave] = total;
	}
	for (int l = WAVES - 1 - wave; l < none; l += WAVES) {
		const int kz = nth(others, l), rz = row_of(kz);
		if (g.dlogits) RowStream<T, CH, 64>::zero((T*)g.dlogits + (long long)rz * g.ldd, g.V, lane);
		if (lane == 0) put_logp(o, rz, kz >= q.T ? q.n + i : i, kz >= q.T ? kz - q.T : kz, false, 0.0, 0.f, 1.f);
	}
	__syncthreads();
	u[0] = part[0][lane & (WAVES - 1)];  // (a wave's sum a lane: all in every lane's registers would be the most that the kernel holds beside its row)
	u[1] = part[1][lane & (WAVES - 1)];
	total = part[2][lane & (WAVES - 1)];
#pragma unroll
	for (int o = WAVES / 2; o > 0; o >>= 1) {
		u[0] += __shfl_xor(u[0], o, 64);
		u[1] += __shfl_xor(u[1], o, 64);
		total += __shfl_xor(total, o, 64);
	}
	if (!q.weight) total = (double)q.n;
	else if (q.total) total = *q.total;
	const double z = pref_margin(q, u[0], u[1]);
	if (threadIdx.x == WAVES * 64 - 1) pref_terms(q, i, z);  // (the last wave: it has the fewest rows)
	if (!g.dlogits) return;
	const float c = pref_slope(q, i, z) * pref_scale(q, total);
	if (wave >= have) return;
	float coef = k >= q.T ? -c : c;
	tile.grad((T*)g.dlogits + (long long)r * g.ldd, g.V, lane, target, xt, m, -coef / s, coef);
	for (int l = wave + WAVES; l < have; l += WAVES) {
		k = nth(counted, l), r = row_of(k), target = of_lane(my_target, k);
		const T* row = (const T*)g.logits + (long long)r * g.ldl;
		const float2 norm = o.norm[r];  // (written by this wave)
		tile.load(row, g.V, lane);
		xt = (float)row[target];
		coef = k >= q.T ? -c : c;
		tile.grad((T*)g.dlogits + (long long)r * g.ldd, g.V, lane, target, xt, norm.x, -coef * norm.y, coef);
	}
}

// ---- policy loss -------------------------------------------------------------------------------------------------------------------------------------------------
constexpr int COUNT_HERE = 1024;
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
	float4* each;      // [A T]: loss, KL, clipped, each times the row's share of the mean; whether it counts
	double* slices;    // [64][4]: sums over the slices of policy_finish_kernel
	float* stats;      // [4]: loss, mean KL, clipped share, counted rows
};
__global__ __launch_bounds__(256) void policy_count_kernel(const Rows g, const Policy p, int lanes) {
	__shared__ int red[8];
	const int lane = threadIdx.x % lanes, teams = 256 / lanes;
	int rows = 0, seqs = 0;
	for (unsigned a = blockIdx.x * teams + threadIdx.x / lanes; a < (unsigned)g.A; a += gridDim.x * teams) {  // (unsigned: what is behind the last may be beyond 2^31)
		int n = 0;
		for (unsigned t = lane; t < (unsigned)g.T; t += lanes) n += counted_target(g, a, t) >= 0;
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
// The counts that a row's share of the mean needs: from policy_count_kernel, or, for at most COUNT_HERE rows (parts = 0), taken by every workgroup for itself, which saves the launch.
struct Counts {
	int total;             // counted rows, or (per_seq) sequences that have any
	const uint8_t* flags;  // LDS: a flag a row, or null
};
__device__ __forceinline__ Counts policy_counts(const Rows& g, const Policy& p, uint8_t* flags, int* red) {
	Counts c = {0, nullptr};
	if (p.parts > 0) {  // the counts of all blocks, by each wave (at most 64 parts)
		const int lane = threadIdx.x & 63;
		c.total = lane < p.parts ? p.part[(p.per_seq ? p.parts : 0) + lane] : 0;
#pragma unroll
		for (int o = 32; o > 0; o >>= 1) c.total += __shfl_xor(c.total, o, 64);
		return c;
	}
	const int R = g.A * g.T;
	for (int r = threadIdx.x; r < R; r += blockDim.x) flags[r] = counted_target(g, r / g.T, r % g.T) >= 0;
	__syncthreads();
	int n = 0;
	for (int r = threadIdx.x; r < R; r += blockDim.x) {
		bool yes = flags[r];
		if (p.per_seq && yes)  // the sequence's first counted row stands for it
			for (int k = r - 1; yes && k >= r - r % g.T; --k) yes = !flags[k];
		n += yes;
	}
#pragma unroll
	for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
	if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
	__syncthreads();
	for (int w = 0; w < (int)(blockDim.x >> 6); ++w) c.total += red[w];
	c.flags = flags;
	return c;
}
// a row's share of the mean, by a team of LANES lanes
template <int LANES>
__device__ __forceinline__ float policy_share(const Rows& g, const Policy& p, const Counts& c, int a, int lane) {
	if (!p.per_seq) return 1.f / (float)c.total;
	int n = 0;
	if (c.flags) {
		for (int t = lane; t < g.T; t += LANES) n += c.flags[a * g.T + t];
#pragma unroll
		for (int o = LANES / 2; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
	} else {
		n = p.len[a];
	}
	return 1.f / ((float)n * (float)c.total);
}
// exp(x) with the range of fp64, up to 2^964, and the accuracy of fp32: no infinity to multiply an advantage of 0 with (a NaN stays one), at a dozen instructions and one fp64 constant
// (the library's functions keep their constants in registers over the whole row: policy rows of 100 columns 19 % slower)
__device__ __forceinline__ double wide_exp(double x) {
	const float k = fminf(fmaxf(rintf((float)x * LOG2E), -1100.f), 900.f);
	float f = (float)fma((double)k, -0.69314718055994530942, x) * LOG2E;
	f = f > 64.f ? 64.f : f;
	return ldexp((double)__builtin_amdgcn_exp2f(f), (int)k);
}
// exp(d) - 1 and exp(d) - d - 1: their series to d^11 where |d| <= 1 (what is left out is below 2^-27 of the sum)
__device__ __forceinline__ void kl_terms(double d, double& rise, double& kl) {
	const float f = (float)d;
	float s = 1.f / 39916800.f;
	s = fmaf(s, f, 1.f / 3628800.f);
	s = fmaf(s, f, 1.f / 362880.f);
	s = fmaf(s, f, 1.f / 40320.f);
	s = fmaf(s, f, 1.f / 5040.f);
	s = fmaf(s, f, 1.f / 720.f);
	s = fmaf(s, f, 1.f / 120.f);
	s = fmaf(s, f, 1.f / 24.f);
	s = fmaf(s, f, 1.f / 6.f);
	s = fmaf(s, f, 0.5f) * f * f;
	const double far = wide_exp(d) - 1.0;
	const bool near = fabsf(f) <= 1.f;
	rise = near ? (double)(f + s) : far;
	kl = near ? (double)s : far - fmin(d, 1e4);  // (infinite at both ends)
}
// The gradient of the whole loss to a row's log-probability.  The ratio and the KL term are exponentials of differences that were formed in fp64; they leave fp32 beyond 88.7, where
// an advantage or a KL coefficient of 0 still makes them nothing.  Products are fp64 up to the one rounding of each result.
struct PolicyRow {
	float loss, kl;  // times the row's share of the mean
	bool whole;      // the unclipped side of the minimum (a NaN takes it and stays one)
};
__device__ __forceinline__ float policy_grad(const Policy& p, int a, int t, double lp, float share, PolicyRow& w) {
	const double q = wide_exp(lp - (double)p.old[a * p.ldold + t]);
	const float adv = p.adv[a * p.lda + t * p.ldt];
	const double held = adv > 0.f ? 1.f + p.hi : 1.f - p.lo;  // the end of the clip range on the side where the minimum takes it
	w.whole = !(adv > 0.f ? q > held : adv < 0.f && q < held);
	double l = -(w.whole ? q : held) * (double)adv, g = w.whole ? l : 0.0;
	w.kl = 0.f;
	if (p.ref) {
		double rise, kl;
		kl_terms((double)p.ref[a * p.ldref + t] - lp, rise, kl);
		if (p.kl_coef != 0.f) {
			l += (double)p.kl_coef * kl;
			g -= (double)p.kl_coef * rise;
		}
		w.kl = (float)(kl * (double)share);
	}
	w.loss = (float)(l * (double)share);
	return (float)(g * (double)share * (double)p.grad_scale);
}
// what one thread of the row writes: its log-probability and its terms of the means
__device__ __forceinline__ void policy_put(const Rows& g, const Policy& p, int r, int a, int t, double lp, float share, const PolicyRow& w) {
	if (p.logp) p.logp[a * p.ldo + t] = (float)lp;
	p.each[r] = make_float4(w.loss, w.kl, w.whole ? 0.f : share, 1.f);
}
__device__ __forceinline__ void policy_put_none(const Rows& g, const Policy& p, int r, int a, int t) {
	if (p.logp) p.logp[a * p.ldo + t] = 0.f;
	p.each[r] = make_float4(0.f, 0.f, 0.f, 0.f);
}
template <typename T, int CH, int THREADS, int NC>
__global__ __launch_bounds__(THREADS) void policy_kernel(const Rows g, const Policy p) {
	__shared__ float red[2 * THREADS / 64];
	__shared__ uint8_t flags[COUNT_HERE];
	__shared__ int counts[THREADS / 64];
	const int r = row_index(g);
	if (r < 0) return;
	const int a = r / g.T, t = r - a * g.T;
	const int target = counted_target(g, a, t);
	T* out = (T*)g.dlogits + (long long)r * g.ldd;
	if (target < 0) {
		if (g.dlogits) RowStream<T, CH, THREADS>::zero(out, g.V, threadIdx.x);
		if (threadIdx.x == 0) policy_put_none(g, p, r, a, t);
		return;
	}
	const T* row = (const T*)g.logits + (long long)r * g.ldl;
	RowTile<T, CH, THREADS, NC> tile;
	tile.load(row, g.V);
	const float xt = (float)row[target], share = policy_share<64>(g, p, policy_counts(g, p, flags, counts), a, threadIdx.x & 63);
	tile.sum(g.V, red);
	const double lp = row_logp(xt, tile.m, tile.s);
	PolicyRow w;
	const float coef = policy_grad(p, a, t, lp, share, w);
	if (threadIdx.x == 0) policy_put(g, p, r, a, t, lp, share, w);
	if (g.dlogits) tile.grad(out, g.V, target, expo(xt, point(tile.m)), coef);
}
template <typename T, int CH, int THREADS>
__global__ __launch_bounds__(THREADS) void policy_long_kernel(const Rows g, const Policy p) {
	__shared__ float red[2 * THREADS / 64];
	__shared__ uint8_t flags[COUNT_HERE];
	__shared__ int counts[THREADS / 64];
	const int r = row_index(g);
	if (r < 0) return;
	const int a = r / g.T, t = r - a * g.T;
	const int target = counted_target(g, a, t);
	T* out = (T*)g.dlogits + (long long)r * g.ldd;
	if (target < 0) {
		if (g.dlogits) RowStream<T, CH, THREADS>::zero(out, g.V, threadIdx.x);
		if (threadIdx.x == 0) policy_put_none(g, p, r, a, t);
		return;
	}
	const T* row = (const T*)g.logits + (long long)r * g.ldl;
	const float xt = (float)row[target], share = policy_share<64>(g, p, policy_counts(g, p, flags, counts), a, threadIdx.x & 63);
	float m, s;
	block_row_sum<T, CH, THREADS>(row, g.V, red, m, s);
	const double lp = row_logp(xt, m, s);
	PolicyRow w;
	const float coef = policy_grad(p, a, t, lp, share, w);
	if (threadIdx.x == 0) policy_put(g, p, r, a, t, lp, share, w);
	if (g.dlogits) RowStream<T, CH, THREADS>::grad(row, out, g.V, threadIdx.x, target, xt, m, -coef / s, coef);
}
template <typename T, int CH, int LANES, int NC>
__global__ __launch_bounds__(256) void policy_team_kernel(const Rows g, const Policy p) {
	const int lane = threadIdx.x % LANES;
	TeamRow<T, CH, LANES, NC> tile;
	Walk<LANES> now(g);
	__shared__ uint8_t flags[COUNT_HERE];
	__shared__ int four[4];
	const Counts shared = policy_counts(g, p, flags, four);
	while (!now.done(g)) {
		const int target = now.target(g);
		const bool counts = target >= 0;
		const T* row = (const T*)g.logits + (long long)now.r * g.ldl;
		T* out = (T*)g.dlogits + (long long)now.r * g.ldd;
		float xt = 0.f, share = 0.f;
		if (counts) {
			tile.load(row, g.V, lane);
			xt = (float)row[target];
			share = policy_share<LANES>(g, p, shared, now.a, lane);
		}
		const Walk<LANES> next = now.next(g);
		if (counts) {
			float m, s;
			tile.sum(g.V, lane, m, s);
			const double lp = row_logp(xt, m, s);
			PolicyRow w;
			const float coef = policy_grad(p, now.a, now.t, lp, share, w);
			if (g.dlogits) tile.grad(out, g.V, lane, target, xt, m, -coef / s, coef);
			if (lane == 0) policy_put(g, p, now.r, now.a, now.t, lp, share, w);
		} else {
			if (g.dlogits) RowStream<T, CH, LANES>::zero(out, g.V, lane);
			if (lane == 0) policy_put_none(g, p, now.r, now.a, now.t);
		}
		now = next;
	}
}
// the sums over a slice of the rows, by workgroup; a second launch adds the slices, unless there is only one
__global__ __launch_bounds__(1024) void policy_finish_kernel(const Rows g, const Policy p) {
	__shared__ double red[48];
	const long long R = (long long)g.A * g.T, slice = (R + gridDim.x - 1) / gridDim.x, first = blockIdx.x * slice, end = min(first + slice, R);
	double l = 0.0, k = 0.0, c = 0.0, n = 0.0;
	for (long long r0 = first + threadIdx.x; r0 < end; r0 += 8 * 1024) {  // eight rows a thread requested at once
		float4 v[8];
#pragma unroll
		for (int i = 0; i < 8; ++i) v[i] = p.each[min(r0 + i * 1024, end - 1)];
#pragma unroll
		for (int i = 0; i < 8; ++i) {
			if (r0 + i * 1024 >= end) continue;
			l += (double)v[i].x;
			k += (double)v[i].y;
			c += (double)v[i].z;
			n += (double)v[i].w;
		}
	}
	sum3_1024(l, k, c, red);
	__syncthreads();
	double none = 0.0, zero = 0.0;
	sum3_1024(n, none, zero, red);
	if (threadIdx.x == 0) {
		const double v[4] = {l, k, c, n};
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			if (gridDim.x == 1) p.stats[i] = (float)v[i];
			else p.slices[4 * blockIdx.x + i] = v[i];
		}
	}
}
__global__ __launch_bounds__(256) void policy_slices_kernel(const Policy p) {
	const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
	double v = p.slices[4 * lane + w];
#pragma unroll
	for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
	if (lane == 0) p.stats[w] = (float)v;
}

// ---- launches ----------------------------------------------------------------------------------------------------------------------------------------------------
// Rows in registers, by workgroup; longer ones take the form that reads a row twice (its second pass comes out of L2 / the memory-side cache).
// (512 lanes with eight vectors each, against 1024 with four: policy step of 315 MB of bf16 logits, 17000 columns 158 and 231 us, 24000 124 and 181, 32700 127 and 164.  1024 with eight
// against reading twice: 40000 columns 170 and 171, 50000 164 and 176, 65000 154 and 176.)
#define NOVIC_ROW_SHAPES(V, REG, LONG)                                                                     \
	if (V <= 512 * CH) { constexpr int TH = 256, NC = 2; REG; }                                              \
	else if (V <= 1024 * CH) { constexpr int TH = 256, NC = 4; REG; }                                        \
	else if (V <= 2048 * CH) { constexpr int TH = 256, NC = 8; REG; }                                        \
	else if (V <= 4096 * CH) { constexpr int TH = 512, NC = 8; REG; }                                        \
	else if (V <= 8192 * CH) { constexpr int TH = 1024, NC = 8; REG; }                                       \
	else { constexpr int TH = 1024; LONG; }
constexpr int SHORT = 128;
// Rows by team: sixteen lanes up to SHORT CH columns (600 bf16 columns: 73 us, by wave 159), a wave with up to MOST vectors a lane beyond
#define NOVIC_TEAM_SHAPES(V, MOST, CALL)                                                                   \
	if (V <= 16 * CH) { constexpr int L = 16, NC = 1; CALL; }                                                \
	else if (V <= 64 * CH) { constexpr int L = 16, NC = 4; CALL; }                                           \
	else if (V <= SHORT * CH) { constexpr int L = 16, NC = SHORT / 16; CALL; }                               \
	else if (MOST == 4 || V <= 4 * 64 * CH) { constexpr int L = 64, NC = 4; CALL; }                          \
	else if (V <= 8 * 64 * CH) { constexpr int L = 64, NC = MOST < 8 ? MOST : 8; CALL; }                     \
	else { constexpr int L = 64, NC = MOST; CALL; }

// Short rows go by team: a workgroup for each is mostly its own start and end ([104857 x 1500] bf16, log-probabilities 84 us by wave, 274 by workgroup; policy with gradient 151 and
// 223; gradient 149 and 211).  Beyond four vectors a lane a workgroup's many registers win where there are gradients to store (4000 columns: 121 and 114 us); without, a wave
// keeps up to sixteen, given rows enough for all waves (6000 columns: 55 and 84 us; at 1500 rows 8.4 and 8.1).
template <int CH>
bool by_team(const Rows& g, bool stores) { return g.V <= 4 * 64 * CH || (!stores && g.V <= 16 * 64 * CH && (long long)g.A * g.T >= 4096); }
template <int LANES>
dim3 team_grid(const Rows& g) { return dim3((unsigned)std::min<long long>(2048, ((long long)g.A * g.T + 256 / LANES - 1) / (256 / LANES))); }
dim3 rows_grid(const Rows& g) {
	const long long R = (long long)g.A * g.T, x = std::min<long long>(R, 1 << 20);
	return dim3((unsigned)x, (unsigned)((R + x - 1) / x));
}
template <typename T, int CH>
void launch_logp(const Rows& g, const LogpOut& o, hipStream_t stream) {
	if constexpr (CH == 1) {
		logp_team_kernel<T, CH, 16, 1><<<team_grid<16>(g), dim3(256), 0, stream>>>(g, o);
	} else if (by_team<CH>(g, false)) {
		NOVIC_TEAM_SHAPES(g.V, 16, (logp_team_kernel<T, CH, L, NC><<<team_grid<L>(g), dim3(256), 0, stream>>>(g, o)))
	} else {
		logp_kernel<T, CH, 256><<<rows_grid(g), dim3(256), 0, stream>>>(g, o);
	}
}
// (gradient by workgroup: 256 lanes, 512 from 1024 CH columns on, 1024 from 4096 CH on: at 6000 bf16 columns 110, 147 and 210 us, at 24000 115, 110 and 115, at 50000 140, 133 and 125)
template <typename T, int CH>
void launch_grad(const Rows& g, const GradIn& in, hipStream_t stream) {
	if constexpr (CH == 1) {
		logp_grad_team_kernel<T, CH, 16><<<team_grid<16>(g), dim3(256), 0, stream>>>(g, in);
	} else {
		if (g.V <= SHORT * CH) logp_grad_team_kernel<T, CH, 16><<<team_grid<16>(g), dim3(256), 0, stream>>>(g, in);
		else if (by_team<CH>(g, true)) logp_grad_team_kernel<T, CH, 64><<<team_grid<64>(g), dim3(256), 0, stream>>>(g, in);
		else if (g.V < 1024 * CH) logp_grad_kernel<T, CH, 256><<<rows_grid(g), dim3(256), 0, stream>>>(g, in);
		else if (g.V < 4096 * CH) logp_grad_kernel<T, CH, 512><<<rows_grid(g), dim3(512), 0, stream>>>(g, in);
		else logp_grad_kernel<T, CH, 1024><<<rows_grid(g), dim3(1024), 0, stream>>>(g, in);
	}
}
template <typename T, int CH>
void launch_policy(const Rows& g, const Policy& p, hipStream_t stream) {
	const dim3 grid = rows_grid(g);
	if constexpr (CH == 1) {
		policy_team_kernel<T, CH, 16, 1><<<team_grid<16>(g), dim3(256), 0, stream>>>(g, p);
	} else if (by_team<CH>(g, true)) {
		NOVIC_TEAM_SHAPES(g.V, 4, (policy_team_kernel<T, CH, L, NC><<<team_grid<L>(g), dim3(256), 0, stream>>>(g, p)))
	} else {
		NOVIC_ROW_SHAPES(g.V, (policy_kernel<T, CH, TH, NC><<<grid, dim3(TH), 0, stream>>>(g, p)), (policy_long_kernel<T, CH, TH><<<grid, dim3(TH), 0, stream>>>(g, p)))
	}
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
constexpr int COUNT_PARTS = 64, SLICES = 64;  // (one wave adds the parts)
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

// Pair by pair where the pairs alone fill the chip (two workgroups of eight waves a unit), a wave's registers hold a row and the row is long enough for a wave; else row by row, with
// the pairs between the two launches over the rows.
constexpr int FUSED_PAIRS = 512, MOST_PAIRS = 1 << 22;  // (a grid's extent in threads is 32 bits)
bool pair_by_pair(const Rows& g, int type) {
	const int ch = type == NOVIC_TYPE_F32 ? 4 : 8;
	return g.A / 2 >= FUSED_PAIRS && g.A / 2 <= MOST_PAIRS && 2 * g.T <= PAIR_ROWS && g.V > 64 * ch && g.V <= PAIR_VECTORS * 64 * ch;
}
// Eight waves, of which two workgroups are resident; sixteen, which read fewer rows twice, for more than sixteen long rows a pair (bf16, 6912 columns, pairs of 2 T rows: T = 32 459 us
// with eight, 396 with sixteen; T = 16 402 and 368; T = 7 302 and 321; T = 3 253 and 363; 2000 columns, T = 16: 228 and 230).
template <typename T, int CH>
void launch_pairs(const Rows& g, const LogpOut& o, const Pref& q, hipStream_t stream) {
	const dim3 grid((unsigned)q.n), eight(8 * 64), sixteen(16 * 64);
	if (g.V <= 4 * 64 * CH) {
		pref_pair_kernel<T, CH, 4, 8><<<grid, eight, 0, stream>>>(g, o, q);
	} else if (g.V <= 8 * 64 * CH) {
		pref_pair_kernel<T, CH, 8, 8><<<grid, eight, 0, stream>>>(g, o, q);
	} else if (g.V <= 12 * 64 * CH) {
		if (2 * g.T <= 16) pref_pair_kernel<T, CH, 12, 8><<<grid, eight, 0, stream>>>(g, o, q);
		else pref_pair_kernel<T, CH, 12, 16><<<grid, sixteen, 0, stream>>>(g, o, q);
	} else {
		if (2 * g.T <= 16) pref_pair_kernel<T, CH, PAIR_VECTORS, 8><<<grid, eight, 0, stream>>>(g, o, q);
		else pref_pair_kernel<T, CH, PAIR_VECTORS, 16><<<grid, sixteen, 0, stream>>>(g, o, q);
	}
}

// workspace: diff [2n T] fp64, each [2][n] fp64, norm [2n T] float2, coef [2n], total fp64, scale
extern "C" uint64_t novic_preference_loss_ws(int n, int T) {
	if (n <= 0 || T <= 0) return 0;
	const uint64_t R = 2ull * n * T;
	return up16(8 * R) + up16(16ull * n) + up16(8 * R) + up16(8ull * n) + 32;
}
extern "C" int novic_preference_loss(const void* logits, int type, int64_t ldl, const void* target, int tok_bytes, int64_t ldt, const uint8_t* pad, int64_t ldp, int n, int T, int V,
                                     const float* ref, int64_t ldref, const float* weight, int kind, double beta, double smoothing, double grad_scale, float* logp, int64_t ldo,
                                     float* margin, void* dlogits, int64_t ldd, float* stats, void* ws, uint64_t ws_bytes, hipStream_t stream) {
	NOVIC_CHECK(n >= 1 && n <= (1 << 29) && T >= 1, "novic_preference_loss: at least one pair and one position, at most 2^29 pairs");
	Rows g = {logits, ldl, dlogits, ldd, target, pad, ldt, ldp, tok_bytes, 2 * n, T, V};
	const char* bad = rows_bad(g, type);
	NOVIC_CHECK(!bad, bad);
	NOVIC_CHECK(ref && stats && ldref >= T && (!logp || ldo >= T), "novic_preference_loss: ref [2n][ldref >= T], stats [3]");
	NOVIC_CHECK(kind == NOVIC_PREF_SIGMOID || kind == NOVIC_PREF_HINGE || kind == NOVIC_PREF_SQUARE, "novic_preference_loss: unknown kind");
	NOVIC_CHECK(beta > 0.0 && beta < INFINITY && smoothing >= 0.0 && smoothing < 0.5 && (smoothing == 0.0 || kind == NOVIC_PREF_SIGMOID), "novic_preference_loss: a finite beta > 0; smoothing in [0, 0.5), with the sigmoid form only");
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
	double* total = (double*)w; w += 16;
	LogpOut o = {};
	o.logp = logp; o.ldo = ldo; o.ref = ref; o.ldref = ldref; o.norm = dlogits ? norm : nullptr;
	Pref q = {diff, weight, n, T, kind, beta, smoothing, grad_scale, margin, coef, each, total, (float*)w, stats};
	if (pair_by_pair(g, type)) {
		if (weight && n > PAIR_WEIGHTS) pref_weight_kernel<<<dim3(1), dim3(1024), 0, stream>>>(q);
		else q.total = nullptr;
		if (type == NOVIC_TYPE_F32) launch_pairs<float, 4>(g, o, q, stream);
		else if (type == NOVIC_TYPE_BF16) launch_pairs<bf16, 8>(g, o, q, stream);
		else launch_pairs<f16, 8>(g, o, q, stream);
		pref_finish_kernel<<<dim3(1), dim3(1024), 0, stream>>>(q);
	} else {
		o.diff = diff;
		NOVIC_ROW_TYPES(type, V, launch_logp, g, o, stream)
		const int lanes = lanes_for(T);
		if ((long long)n * lanes <= 2048) {  // two rounds of one workgroup: shorter than a second launch
			pref_all_kernel<<<dim3(1), dim3(1024), 0, stream>>>(q, lanes);
		} else {
			pref_each_kernel<<<dim3((unsigned)(((long long)n * lanes + 255) / 256)), dim3(256), 0, stream>>>(q, lanes);
			pref_finish_kernel<<<dim3(1), dim3(1024), 0, stream>>>(q);
		}
		if (dlogits) {
			GradIn in = {};
			in.norm = norm; in.grad = coef; in.lda = 1; in.ldt = 0; in.scale = q.scale;
			NOVIC_ROW_TYPES(type, V, launch_grad, g, in, stream)
		}
	}
	NOVIC_LAUNCH_CHECK();
	return 0;
}

// workspace: len [A], part [2][64], slices [64][4] fp64, each [A T] float4
extern "C" uint64_t novic_policy_loss_ws(int A, int T) {
	if (A <= 0 || T <= 0) return 0;
	return up16(4ull * A) + up16(8 * COUNT_PARTS) + 32 * SLICES + 16ull * A * T;
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
	p.slices = (double*)w; w += 32 * SLICES;
	p.each = (float4*)w;
	const bool counted = (long long)A * T > COUNT_HERE;
	p.parts = counted ? count_parts(A, T) : 0;
	p.stats = stats;
	if (counted) policy_count_kernel<<<dim3(p.parts), dim3(256), 0, stream>>>(g, p, lanes_for(T));
	NOVIC_ROW_TYPES(type, V, launch_policy, g, p, stream)
	// one workgroup reads its rows' terms at some 50 GB/s: beyond 8192 rows (a batch of loads a thread) 64 of them and one launch more are shorter
	const bool sliced = (long long)A * T > 8192;
	policy_finish_kernel<<<dim3(sliced ? SLICES : 1), dim3(1024), 0, stream>>>(g, p);
	if (sliced) policy_slices_kernel<<<dim3(1), dim3(256), 0, stream>>>(p);
	NOVIC_LAUNCH_CHECK();
	return 0;
}
