// LayerNorm that keeps its row statistics, forward and backward, with the reduction of both affine gradients in a fixed order.
//
//   forward    mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), y = (x - mu) rstd gamma + beta
//   backward   g = dy gamma, xhat = (x - mu) rstd:  dx = dx_in + rstd (g - mean(g) - xhat mean(g xhat));  dgamma = sum_rows dy xhat, dbeta = sum_rows dy
//
// HBM-bound both ways: each element is read once and written once, the row lives in registers between its statistics and its output (the two-pass variance costs no second
// read), statistics and sums in fp32.  A row belongs to a team of 16, 64 or 256 lanes, the smallest that holds it in about four vectors a lane, or of 512, whose lanes take up to
// eight (with 1024 lanes a lane has 128 registers: 5 % faster backward at 16384 columns, but one type's form spills, and 6 to 40 % slower forward).  What is read once is loaded, and
// gradients are stored, past the caches.  MI355X: forward [57344 x 512] fp32 -> bf16 30.4 us (5.8 TB/s), [65792 x 1280] bf16 66 us (5.1); backward [65792 x 1280] bf16 with both
// affine gradients and the residual's added 121 us (5.6 TB/s, of it 5 us in the reduction of the partial rows; without those hints 132).
#include "novic_hip.h"
#include "rowvec.hpp"

namespace {

// sums of one or two values over a team; teams of more than a wave go through LDS (scratch: two floats per wave, double-buffered by `turn` so that one barrier a use is enough)
template <int LANES>
__device__ __forceinline__ void team_sum2(float& a, float& b, float* scratch, int& turn) {
	a = team_sum<(LANES < 64 ? LANES : 64)>(a);
	b = team_sum<(LANES < 64 ? LANES : 64)>(b);
	if constexpr (LANES > 64) {
		constexpr int W = LANES / 64;
		float* s = scratch + (turn & 1) * 2 * W;
		turn ^= 1;
		const int w = threadIdx.x >> 6;
		if ((threadIdx.x & 63) == 0) {
			s[2 * w] = a;
			s[2 * w + 1] = b;
		}
		__syncthreads();
		a = team_sum<W>(s[2 * (threadIdx.x & (W - 1))]);
		b = team_sum<W>(s[2 * (threadIdx.x & (W - 1)) + 1]);
	}
}

// waves a SIMD: what the grid of plan() counts on
constexpr int fwd_waves(int lanes, int held) { return held <= 24 && (lanes <= 256 || held <= 16) ? 4 : lanes <= 256 ? 3 : 2; }
template <typename XT, typename YT, int CH, int LANES, int NC>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256, fwd_waves(LANES, NC * CH)) void layernorm_stats_fwd_kernel(const XT* x, long long ldx, const float* __restrict__ gamma,
                                                                                       const float* __restrict__ beta, YT* y, long long ldy,
                                                                                       float* __restrict__ mean_out, float* __restrict__ rstd_out, int rows, int E, float eps) {
	constexpr int THREADS = LANES > 256 ? LANES : 256, TEAMS = THREADS / LANES;
	__shared__ float scratch[LANES > 64 ? 4 * (LANES / 64) : 1];
	const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
	int es[NC], turn = 0;
	RawVec<float, CH> gm[NC], bt[NC];
#pragma unroll
	for (int c = 0; c < NC; ++c) {
		const int e0 = (c * LANES + lane) * CH;
		es[c] = c < NC - 1 ? e0 : min(e0, E - CH);  // (all vectors but a lane's last lie inside the row: the plan takes the smallest NC)
		gm[c] = load_vec<float, CH>(elem(gamma, es[c]));
		if (beta) bt[c] = load_vec<float, CH>(elem(beta, es[c]));
	}
	const float inv = 1.f / (float)E;
	const int stride = gridDim.x * TEAMS;
	auto load = [&](RawVec<XT, CH> (&raw)[NC], int of) {
		const int row = LANES < 64 ? of : __builtin_amdgcn_readfirstlane(of);  // (the same for a wave)
#pragma unroll
		for (int c = 0; c < NC; ++c) raw[c] = load_once<XT, CH>(elem(x + (long long)row * ldx, es[c]));
	};
	RawVec<XT, CH> raw[NC], next[NC];
	const int first = blockIdx.x * TEAMS + team;
	if (first < rows) load(raw, first);
	// (teams of more than a wave have a block of their own, so the rows of a block and with them the barriers in team_sum2 are the same for all its threads.  What is left is counted
	// down: the row behind the last, up to a stride of 16384 beyond 2^31, is no int)
	for (int left = rows - first; left > 0; left -= stride) {
		const int row0 = rows - left, row = LANES < 64 ? row0 : __builtin_amdgcn_readfirstlane(row0);
		load(next, rows - max(left - stride, 1));  // requested before this row is reduced
		float s = 0.f, q = 0.f, off = 0.f, none = 0.f;
#pragma unroll
		for (int c = 0; c < NC; ++c) {
#pragma unroll
			for (int i = 0; i < CH; ++i)
				if (c < NC - 1 || es[c] + i >= (c * LANES + lane) * CH) s += raw[c].get(i);
			if constexpr (NC * CH > 16) forget(raw[c]);  // (the deviations of a long row are formed where they are used: held, they would cost the registers of a resident workgroup)
		}
		team_sum2<LANES>(s, none, scratch, turn);
		// The first mean is off by the sum's rounding, which a row far from zero would carry into every element: the deviations' own mean `off` corrects it, at no extra reduction.
		float mean = s / (float)E;
#pragma unroll
		for (int c = 0; c < NC; ++c) {
#pragma unroll
			for (int i = 0; i < CH; ++i) {
				const float d = raw[c].get(i) - mean;
				if (c < NC - 1 || es[c] + i >= (c * LANES + lane) * CH) {
					q += d * d;
					off += d;
				}
			}
			if constexpr (NC * CH > 16) forget(raw[c]);
		}
		team_sum2<LANES>(q, off, scratch, turn);
		off *= inv;
		const float first_mean = mean;
		mean += off;
		const float var = q * inv - off * off;
		const float rstd = rsqrtf((var < 0.f ? 0.f : var) + eps);  // (a NaN stays one)
		if (lane == 0) {
			if (mean_out) mean_out[row] = mean;
			if (rstd_out) rstd_out[row] = rstd;
		}
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			if (c == NC - 1 && (c * LANES + lane) * CH >= E) continue;
			float o[CH];
#pragma unroll
			for (int i = 0; i < CH; ++i) {
				float t = ((raw[c].get(i) - first_mean) - off) * rstd * gm[c].get(i);
				if (beta) t += bt[c].get(i);
				o[i] = t;
			}
			store_own<false>(y + (long long)row * ldy, es[c], (c * LANES + lane) * CH, o);
		}
#pragma unroll
		for (int c = 0; c < NC; ++c) raw[c] = next[c];
	}
}

// The affine gradients: a lane owns the same columns in every row, so it adds them up in registers over all rows of its team; a block adds its teams through LDS and writes
// ONE partial row of each gradient, layernorm_stats_reduce_kernel adds the partial rows in their order.  No atomics: the same inputs give the same bits.
template <typename XT, typename YT, int CH, int LANES, int NC>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void layernorm_stats_bwd_kernel(const YT* dy, long long lddy, const XT* x, long long ldx,
                                                                                       const float* gamma, const float* mean, const float* rstd,
                                                                                       const XT* dx_in, long long ldi, XT* dx, long long lddx,
                                                                                       float* __restrict__ part_gamma, float* __restrict__ part_beta, int rows, int E, int accumulate) {
	constexpr int THREADS = LANES > 256 ? LANES : 256, TEAMS = THREADS / LANES;
	__shared__ float scratch[LANES > 64 ? 4 * (LANES / 64) : 1];
	__shared__ float fold[TEAMS > 1 ? THREADS * CH : 1];
	// The next row is requested before the current one is reduced: a team always has a row's worth of loads in flight.  Not in teams of 512 lanes, whose registers hold
	// one row only: they load the row where it is used, gamma with it (out of the cache, where all teams keep it).
	constexpr bool AHEAD = LANES < 512;
	const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
	int es[NC], turn = 0;
	RawVec<float, CH> gm[NC];
	float dg[NC][CH], db[NC][CH];
#pragma unroll
	for (int c = 0; c < NC; ++c) {
		es[c] = c < NC - 1 ? (c * LANES + lane) * CH : min((c * LANES + lane) * CH, E - CH);
		if (AHEAD) gm[c] = load_vec<float, CH>(elem(gamma, es[c]));
#pragma unroll
		for (int i = 0; i < CH; ++i) dg[c][i] = db[c][i] = 0.f;
	}
	const float inv = 1.f / (float)E;
	struct Row {
		RawVec<XT, CH> x[NC], in[NC];
		RawVec<YT, CH> dy[NC];
		float mu, rs;
	};
	auto load = [&](Row& r, int of) {
		const int row = LANES < 64 ? of : __builtin_amdgcn_readfirstlane(of);  // (the same for a wave)
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			r.x[c] = load_once<XT, CH>(elem(x + (long long)row * ldx, es[c]));
			r.dy[c] = load_once<YT, CH>(elem(dy + (long long)row * lddy, es[c]));
			if (AHEAD && dx_in) r.in[c] = load_once<XT, CH>(elem(dx_in + (long long)row * ldi, es[c]));
		}
		r.mu = mean[row];
		r.rs = rstd[row];
	};
	const int stride = gridDim.x * TEAMS;
	int row = blockIdx.x * TEAMS + team;
	if (LANES >= 64) row = __builtin_amdgcn_readfirstlane(row);
	Row cur;
	if (AHEAD && row < rows) load(cur, row);
	for (int left = rows - row; left > 0; left -= stride) {  // (counted down as in the forward kernel)
		row = rows - left;
		Row nxt;
		if (AHEAD) load(nxt, rows - max(left - stride, 1));
		else load(cur, row);
		float s1 = 0.f, s2 = 0.f;
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			if (!AHEAD) {
				asm volatile("" ::: "memory");  // (vector by vector: all of gamma at once has no room)
				__builtin_amdgcn_sched_barrier(0);
				gm[c] = load_vec<float, CH>(elem(gamma, es[c]));
			}
#pragma unroll
			for (int i = 0; i < CH; ++i)
				if (c < NC - 1 || es[c] + i >= (c * LANES + lane) * CH) {
					const float g = cur.dy[c].get(i) * gm[c].get(i);
					s1 += g;
					s2 += g * ((cur.x[c].get(i) - cur.mu) * cur.rs);
				}
		}
		team_sum2<LANES>(s1, s2, scratch, turn);
		s1 *= inv;
		s2 *= inv;
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			forget(cur.x[c]);  // (xhat and g are formed again: two registers an element less over the reduction)
			forget(cur.dy[c]);
			if (c == NC - 1 && (c * LANES + lane) * CH >= E) continue;
			if (!AHEAD) {
				asm volatile("" ::: "memory");
				__builtin_amdgcn_sched_barrier(0);
				gm[c] = load_vec<float, CH>(elem(gamma, es[c]));
				if (dx_in) cur.in[c] = load_once<XT, CH>(elem(dx_in + (long long)row * ldi, es[c]));
			}
			float o[CH];
#pragma unroll
			for (int i = 0; i < CH; ++i) {
				const float d = cur.dy[c].get(i), xh = (cur.x[c].get(i) - cur.mu) * cur.rs;
				if (c < NC - 1 || es[c] + i >= (c * LANES + lane) * CH) {
					dg[c][i] += d * xh;
					db[c][i] += d;
				}
				float t = cur.rs * (d * gm[c].get(i) - s1 - xh * s2);
				if (dx_in) t += cur.in[c].get(i);
				o[i] = t;
			}
			store_own<true>(dx + (long long)row * lddx, es[c], (c * LANES + lane) * CH, o);
		}
		if (AHEAD) cur = nxt;
	}
	auto put = [&](const float (&acc)[NC][CH], float* part) {
		if (!part) return;
		float* out = part + (long long)blockIdx.x * E;
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			float t[CH];
#pragma unroll
			for (int i = 0; i < CH; ++i) t[i] = acc[c][i];
			if constexpr (TEAMS > 1) {
				__syncthreads();
#pragma unroll
				for (int i = 0; i < CH; ++i) fold[i * THREADS + threadIdx.x] = t[i];
				__syncthreads();
				if (team == 0) {
#pragma unroll
					for (int k = 1; k < TEAMS; ++k)
#pragma unroll
						for (int i = 0; i < CH; ++i) t[i] += fold[i * THREADS + k * LANES + lane];
				}
			}
			if (team == 0) {
#pragma unroll
				for (int i = 0; i < CH; ++i) {
					const int e = es[c] + i;
					if (c < NC - 1 || e >= (c * LANES + lane) * CH) out[e] = accumulate ? out[e] + t[i] : t[i];
				}
			}
		}
	};
	put(dg, part_gamma);
	put(db, part_beta);
}

// out[e] (+)= sum over the partial rows of part[row][e], in their order: 32 columns a block, 32 groups of rows, the groups' sums added in order.  blockIdx.y: which gradient.
__global__ __launch_bounds__(1024) void layernorm_stats_reduce_kernel(const float* __restrict__ part_gamma, const float* __restrict__ part_beta, float* __restrict__ dgamma,
                                                                      float* __restrict__ dbeta, int parts, int E, int accumulate) {
	__shared__ float sum[32][33];
	const float* part = blockIdx.y == 0 ? part_gamma : part_beta;
	float* out = blockIdx.y == 0 ? dgamma : dbeta;
	if (!out) return;  // uniform over the block
	const int col = threadIdx.x & 31, grp = threadIdx.x >> 5, e = blockIdx.x * 32 + col;
	float t = 0.f;
	for (int r0 = grp; e < E && r0 < parts; r0 += 8 * 32) {  // eight partial rows a thread requested at once
		float v[8];
#pragma unroll
		for (int k = 0; k < 8; ++k) v[k] = part[(long long)min(r0 + k * 32, parts - 1) * E + e];
#pragma unroll
		for (int k = 0; k < 8; ++k) t += r0 + k * 32 < parts ? v[k] : 0.f;
	}
	sum[grp][col] = t;
	__syncthreads();
	if (grp == 0 && e < E) {
		t = 0.f;
#pragma unroll
		for (int k = 0; k < 32; ++k) t += sum[k][col];
		out[e] = accumulate ? out[e] + t : t;
	}
}

struct Plan {
	int lanes, chunks, blocks;
};
// ch: elements of a lane's vector
Plan plan(int rows, int E, int ch, bool bwd) {
	Plan p;
	// Forward: sixteen lanes up to four vectors each ([200000 x 100] fp32 -> bf16: 25 us, by wave 60), a wave up to five fp32 vectors ([65792 x 1280]: 95 us, with 256 lanes 129; more would spill).
	// Backward: sixteen lanes up to 256 columns (the same rows: 49 and 86 us; at 512 bf16 columns 51 and 39), a wave up to four vectors a lane.
	const int narrow = bwd ? 256 : 64 * ch, wide = ch == 4 && !bwd ? 1280 : 256 * ch;
	p.lanes = E <= narrow ? 16 : E <= wide ? 64 : E <= 1024 * ch ? 256 : 512;
	p.chunks = (E + p.lanes * ch - 1) / (p.lanes * ch);
	const int teams = p.lanes > 256 ? 1 : 256 / p.lanes;
	// Forward: as many workgroups as are resident at once, up to four a unit (more are slower: 1024 of them 30.2 us, 2048 31.8 on [57344 x 512]; a part of them left over for a second
	// round is worse).  Backward: as many as are resident, two a unit or one: each leaves a partial row of both gradients behind.  A handful of rows is one workgroup's business,
	// which needs no second launch (16 rows of 512: 9.4 us a call, with it 13.5).
	const int held = p.chunks * ch;
	int most;
	if (bwd) most = rows <= 4 * teams ? 1 : p.lanes > 256 && held > 16 ? 256 : 512;
	else most = p.lanes > 256 ? (held <= 16 ? 512 : 256) : held <= 24 ? 1024 : 768;
	p.blocks = (int)std::min<long long>(most, ((long long)rows + teams - 1) / teams);
	return p;
}
int chunk_elems(int x_type, int y_type, int E) { return E < 8 ? 1 : (x_type != NOVIC_TYPE_F32 && y_type != NOVIC_TYPE_F32) ? 8 : 4; }

// (a shape that no width of this vector length asks for is not compiled)
#define NOVIC_LN_CASE(LANES, NC, CALL)                                                         \
	if constexpr ((NC - 1) * LANES * CH < 16384 && (CH > 1 || (LANES == 16 && NC == 1))) {                    \
		if (p.lanes == LANES && p.chunks == NC) { constexpr int L = LANES, N = NC; CALL; }          \
	}
#define NOVIC_LN_SHAPES(CALL)                                                                                                                             \
	NOVIC_LN_CASE(16, 1, CALL) NOVIC_LN_CASE(16, 2, CALL) NOVIC_LN_CASE(16, 3, CALL) NOVIC_LN_CASE(16, 4, CALL)                                           \
	NOVIC_LN_CASE(64, 1, CALL) NOVIC_LN_CASE(64, 2, CALL) NOVIC_LN_CASE(64, 3, CALL) NOVIC_LN_CASE(64, 4, CALL)                                           \
	NOVIC_LN_CASE(256, 2, CALL) NOVIC_LN_CASE(256, 3, CALL) NOVIC_LN_CASE(256, 4, CALL)                                                                    \
	NOVIC_LN_CASE(512, 3, CALL) NOVIC_LN_CASE(512, 4, CALL) NOVIC_LN_CASE(512, 5, CALL) NOVIC_LN_CASE(512, 6, CALL) NOVIC_LN_CASE(512, 7, CALL) NOVIC_LN_CASE(512, 8, CALL)

bool types_ok(int x_type, int y_type) {
	return x_type >= NOVIC_TYPE_F32 && x_type <= NOVIC_TYPE_F16 && y_type >= NOVIC_TYPE_F32 && y_type <= NOVIC_TYPE_F16 && (x_type == y_type || x_type == NOVIC_TYPE_F32);
}

template <typename XT, typename YT, int CH>
void launch_fwd(const Plan& p, const void* x, long long ldx, const float* gamma, const float* beta, void* y, long long ldy, float* mean, float* rstd, int rows, int E, float eps,
                hipStream_t stream) {
#define NOVIC_LN_FWD (layernorm_stats_fwd_kernel<XT, YT, CH, L, N><<<dim3(p.blocks), dim3(L > 256 ? L : 256), 0, stream>>>((const XT*)x, ldx, gamma, beta, (YT*)y, ldy, mean, rstd, rows, E, eps))
	NOVIC_LN_SHAPES(NOVIC_LN_FWD)
	if constexpr (CH == 4) { NOVIC_LN_CASE(64, 5, NOVIC_LN_FWD) }
}
template <typename XT, typename YT, int CH>
void launch_bwd(const Plan& p, const void* dy, long long lddy, const void* x, long long ldx, const float* gamma, const float* mean, const float* rstd, const void* dx_in, long long ldi,
                void* dx, long long lddx, float* pg, float* pb, int rows, int E, int accumulate, hipStream_t stream) {
	NOVIC_LN_SHAPES((layernorm_stats_bwd_kernel<XT, YT, CH, L, N><<<dim3(p.blocks), dim3(L > 256 ? L : 256), 0, stream>>>((const YT*)dy, lddy, (const XT*)x, ldx, gamma,
	                                    mean, rstd, (const XT*)dx_in, ldi, (XT*)dx, lddx, pg, pb, rows, E, accumulate)))
}
#define NOVIC_LN_TYPES(FN, ...)                                                                                             \
	if (E < 8) { /* narrower than a vector: single elements */                                                             \
		if (x_type == NOVIC_TYPE_F32) NOVIC_TYPE_SWITCH(y_type, YT, (FN<float, YT, 1>(__VA_ARGS__)))                          \
		else if (x_type == NOVIC_TYPE_BF16) FN<bf16, bf16, 1>(__VA_ARGS__);                                                   \
		else FN<f16, f16, 1>(__VA_ARGS__);                                                                                    \
	} else if (x_type == NOVIC_TYPE_F32) NOVIC_TYPE_SWITCH(y_type, YT, (FN<float, YT, 4>(__VA_ARGS__)))                       \
	else if (x_type == NOVIC_TYPE_BF16) FN<bf16, bf16, 8>(__VA_ARGS__);                                                       \
	else FN<f16, f16, 8>(__VA_ARGS__);

}  // namespace

extern "C" int novic_layernorm_stats_fwd(const void* x, int x_type, int64_t ldx, const float* gamma, const float* beta, void* y, int y_type, int64_t ldy, float* mean, float* rstd,
                                         int rows, int E, float eps, hipStream_t stream) {
	NOVIC_CHECK(types_ok(x_type, y_type), "novic_layernorm_stats_fwd: y has x's type, or any type where x is fp32");
	NOVIC_CHECK(E >= 1 && E <= 16384, "novic_layernorm_stats_fwd: 1 <= E <= 16384");
	NOVIC_CHECK(rows >= 0 && (rows <= 1 || (ldx >= E && ldy >= E)), "novic_layernorm_stats_fwd: rows >= 0, leading dimensions >= E");
	if (rows == 0) return 0;
	NOVIC_CHECK(x && gamma && y, "novic_layernorm_stats_fwd: null pointer");
	NOVIC_APART("novic_layernorm_stats_fwd", NOVIC_SPANS({y, rows, E * type_bytes(y_type), ldy * type_bytes(y_type)}, {mean, 1, 4LL * rows, 0}, {rstd, 1, 4LL * rows, 0}),
	            NOVIC_SPANS({gamma, 1, 4LL * E, 0}, {beta, 1, 4LL * E, 0}, {x_type == y_type ? nullptr : x, rows, E * type_bytes(x_type), ldx * type_bytes(x_type)}),
	            NOVIC_SPANS({x_type == y_type ? x : nullptr, rows, E * type_bytes(x_type), ldx * type_bytes(x_type)}))
	const Plan p = plan(rows, E, chunk_elems(x_type, y_type, E), false);
	NOVIC_LN_TYPES(launch_fwd, p, x, ldx, gamma, beta, y, ldy, mean, rstd, rows, E, eps, stream)
	NOVIC_LAUNCH_CHECK();
	return 0;
}

extern "C" uint64_t novic_layernorm_stats_bwd_ws(int rows, int E, int x_type, int y_type) {
	if (rows <= 0 || E < 1 || E > 16384 || !types_ok(x_type, y_type)) return 0;
	const Plan p = plan(rows, E, chunk_elems(x_type, y_type, E), true);
	return p.blocks == 1 ? 0 : (uint64_t)p.blocks * E * 8;
}

extern "C" int novic_layernorm_stats_bwd(const void* dy, int y_type, int64_t lddy, const void* x, int x_type, int64_t ldx, const float* gamma, const float* mean, const float* rstd,
                                         const void* dx_in, int64_t ldi, void* dx, int64_t lddx, float* dgamma, float* dbeta, int accumulate, int rows, int E, void* ws,
                                         uint64_t ws_bytes, hipStream_t stream) {
	NOVIC_CHECK(types_ok(x_type, y_type), "novic_layernorm_stats_bwd: dy has x's type, or any type where x is fp32");
	NOVIC_CHECK(E >= 1 && E <= 16384, "novic_layernorm_stats_bwd: 1 <= E <= 16384");
	NOVIC_CHECK(rows >= 0 && (rows <= 1 || (ldx >= E && lddy >= E && lddx >= E && (!dx_in || ldi >= E))), "novic_layernorm_stats_bwd: rows >= 0, leading dimensions >= E");
	NOVIC_CHECK(rows == 0 || (dy && x && gamma && mean && rstd && dx), "novic_layernorm_stats_bwd: null pointer");
	const long long bx = type_bytes(x_type), by = type_bytes(y_type);
	NOVIC_APART("novic_layernorm_stats_bwd", NOVIC_SPANS({dx, rows, E * bx, lddx * bx}, {dgamma, 1, 4LL * E, 0}, {dbeta, 1, 4LL * E, 0}),
	            NOVIC_SPANS({gamma, 1, 4LL * E, 0}, {mean, 1, 4LL * rows, 0}, {rstd, 1, 4LL * rows, 0}, {x_type == y_type ? nullptr : dy, rows, E * by, lddy * by}),
	            NOVIC_SPANS({x, rows, E * bx, ldx * bx}, {dx_in, rows, E * bx, ldi * bx}, {x_type == y_type ? dy : nullptr, rows, E * by, lddy * by}))
	const Plan p = plan(rows, E, chunk_elems(x_type, y_type, E), true);
	const bool affine = dgamma || dbeta;
	const bool direct = p.blocks == 1;  // one block: its sums are the gradients, no second launch
	NOVIC_CHECK(!affine || rows == 0 || direct || (ws && ws_bytes >= (uint64_t)p.blocks * E * 8), "novic_layernorm_stats_bwd: the workspace is smaller than novic_layernorm_stats_bwd_ws says");
	float* pg = !dgamma ? nullptr : direct ? dgamma : (float*)ws;
	float* pb = !dbeta ? nullptr : direct ? dbeta : (float*)ws + (size_t)p.blocks * E;
	if (rows > 0) {
		NOVIC_LN_TYPES(launch_bwd, p, dy, lddy, x, ldx, gamma, mean, rstd, dx_in, ldi, dx, lddx, pg, pb, rows, E, direct && accumulate, stream)
	}
	if (affine && (rows == 0 ? !accumulate : !direct))  // (no rows: the sums are zero)
		layernorm_stats_reduce_kernel<<<dim3((E + 31) / 32, 2), dim3(1024), 0, stream>>>(pg, pb, dgamma, dbeta, rows == 0 ? 0 : p.blocks, E, accumulate);
	NOVIC_LAUNCH_CHECK();
	return 0;
}
