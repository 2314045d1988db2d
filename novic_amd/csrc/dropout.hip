// Dropout from a counter-based generator, with a mask that is never stored, and its backward pass.
//
//   keep(i) = u16(i) >= thr, thr = round(65536 p);   y[i] = (keep(i) ? x[i] * 65536 / (65536 - thr) : 0) (+ resid[i]);   dx[i] = keep(i) ? dy[i] * 65536 / (65536 - thr) : 0
//
// u16(i): Philox4x32-10 with the seed as key and the counter (block low, block high, site, step), block = i / 8, i = the element's index in the row-major [rows][cols] matrix
// without its row padding: a block's 128 bits are the eight 16-bit numbers of its elements, the low half of a word first.  The mask is a function of (seed, site, step, i) alone:
// the backward pass draws it again.  `step` may be a device scalar, so that a replayed graph draws a new mask each time.  The scale uses the probability that 16 bits hold,
// which keeps the expectation exact.
//
// HBM-bound: one generator block (20 32 x 32 -> 64-bit multiplies) serves one 16-byte vector of 16-bit elements.  MI355X: [57344 x 512] bf16 + fp32 residual -> fp32 54 us
// (294 MB, 5.5 TB/s).
#include "novic_hip.h"
#include "rowvec.hpp"

namespace {

struct Args {
	const void* x;
	void* y;
	const void* resid;
	long long ldx, ldy, ldr;
	long long rows, cols;
	const long long* step;  // device scalar (low 32 bits count) or null: 0
	uint32_t thr, seed_lo, seed_hi, site;
	float scale;
};

__device__ __forceinline__ void mask8(const Args& g, uint32_t step, unsigned long long block, bool (&keep)[8]) {
	const Philox4 r = philox4x32_10((uint32_t)block, (uint32_t)(block >> 32), g.site, step, g.seed_lo, g.seed_hi);
	const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		keep[2 * i] = (w[i] & 0xffffu) >= g.thr;
		keep[2 * i + 1] = (w[i] >> 16) >= g.thr;
	}
}
// (a dropped element is a zero whatever it was: an infinity or a NaN does not pass)
__device__ __forceinline__ float dropped(const Args& g, bool keep, float x) { return keep ? x * g.scale : 0.f; }

// no row padding: the matrix is one run of elements; a thread takes whole generator blocks
template <typename XT, typename YT, bool RESID>
__global__ __launch_bounds__(256) void dropout_flat_kernel(const Args g) {
	const long long n = g.rows * g.cols, blocks = n >> 3;
	const uint32_t step = g.step ? (uint32_t)*g.step : 0u;
	const XT* x = (const XT*)g.x;
	YT* y = (YT*)g.y;
	const YT* resid = (const YT*)g.resid;
	const long long first = (long long)blockIdx.x * 256 + threadIdx.x, stride = (long long)gridDim.x * 256;
	for (long long b = first; b < blocks; b += stride) {
		const RawVec<XT, 8> v = load_vec<XT, 8>(x + 8 * b);
		RawVec<YT, 8> r;
		float o[8];
		if (RESID) r = load_vec<YT, 8>(resid + 8 * b);
		bool keep[8];
		mask8(g, step, b, keep);
#pragma unroll
		for (int i = 0; i < 8; ++i) {
			float t = dropped(g, keep[i], v.get(i));
			if (RESID) t += r.get(i);
			o[i] = t;
		}
		store_vec<false>(y + 8 * b, o);
	}
	if (first == 0 && (n & 7)) {  // the last, partial block
		bool keep[8];
		mask8(g, step, blocks, keep);
		for (int i = 0; i < (int)(n & 7); ++i) {
			const long long e = 8 * blocks + i;
			float t = dropped(g, keep[i], (float)x[e]);
			if (RESID) t += (float)resid[e];
			y[e] = (YT)t;
		}
	}
}

// rows with padding between them: a thread takes one generator block of one row; a block that spans the end of a row is drawn once for each of the two
template <typename XT, typename YT, bool RESID>
__global__ __launch_bounds__(256) void dropout_rows_kernel(const Args g) {
	const uint32_t step = g.step ? (uint32_t)*g.step : 0u;
	for (long long row = blockIdx.y; row < g.rows; row += gridDim.y) {
		const XT* x = (const XT*)g.x + row * g.ldx;
		YT* y = (YT*)g.y + row * g.ldy;
		const YT* resid = (const YT*)g.resid + row * g.ldr;
		const long long base = row * g.cols, end = base + g.cols;
		for (long long b = (base >> 3) + (long long)blockIdx.x * 256 + threadIdx.x; 8 * b < end; b += (long long)gridDim.x * 256) {
			bool keep[8];
			mask8(g, step, b, keep);
			const long long e = 8 * b - base;  // column of the block's first element: below zero where the block began in the row before
			if (e >= 0 && e + 8 <= g.cols) {
				const RawVec<XT, 8> v = load_vec<XT, 8>(x + e);
				RawVec<YT, 8> r;
				float o[8];
				if (RESID) r = load_vec<YT, 8>(resid + e);
#pragma unroll
				for (int i = 0; i < 8; ++i) {
					float t = dropped(g, keep[i], v.get(i));
					if (RESID) t += r.get(i);
					o[i] = t;
				}
				store_vec<false>(y + e, o);
			} else {
#pragma unroll
				for (int i = 0; i < 8; ++i) {
					if (e + i < 0 || e + i >= g.cols) continue;
					float t = dropped(g, keep[i], (float)x[e + i]);
					if (RESID) t += (float)resid[e + i];
					y[e + i] = (YT)t;
				}
			}
		}
	}
}

template <typename XT, typename YT>
void launch(const Args& g, hipStream_t stream) {
	const bool flat = g.rows == 1 || (g.ldx == g.cols && g.ldy == g.cols && (!g.resid || g.ldr == g.cols));
	if (flat) {
		// a vector a thread and no loop, as far as the grid goes: 41.5 us on 117 MB of bf16 (5.7 TB/s), against 45.6 with 2048 workgroups that walk over it
		const int grid = (int)std::min<long long>(1 << 22, std::max<long long>(1, (g.rows * g.cols / 8 + 255) / 256));
		if (g.resid) dropout_flat_kernel<XT, YT, true><<<dim3(grid), dim3(256), 0, stream>>>(g);
		else dropout_flat_kernel<XT, YT, false><<<dim3(grid), dim3(256), 0, stream>>>(g);
	} else {
		const dim3 grid((unsigned)std::min<long long>(64, (g.cols / 8 + 1 + 255) / 256), (unsigned)std::min<long long>(4096, g.rows));
		if (g.resid) dropout_rows_kernel<XT, YT, true><<<grid, dim3(256), 0, stream>>>(g);
		else dropout_rows_kernel<XT, YT, false><<<grid, dim3(256), 0, stream>>>(g);
	}
}

}  // namespace

extern "C" int novic_dropout(const void* x, int x_type, int64_t ldx, const void* resid, int64_t ldr, void* y, int y_type, int64_t ldy, int64_t rows, int64_t cols, double p, uint64_t seed,
                             uint32_t site, const int64_t* step, hipStream_t stream) {
	NOVIC_CHECK(x_type >= NOVIC_TYPE_F32 && x_type <= NOVIC_TYPE_F16 && y_type >= NOVIC_TYPE_F32 && y_type <= NOVIC_TYPE_F16, "novic_dropout: unknown element type");
	NOVIC_CHECK(x_type == y_type || x_type == NOVIC_TYPE_F32 || y_type == NOVIC_TYPE_F32, "novic_dropout: the two types are equal, or one of them is fp32");
	NOVIC_CHECK(p >= 0.0 && p <= 1.0, "novic_dropout: 0 <= p <= 1");
	NOVIC_CHECK(rows >= 0 && cols >= 0 && (rows <= 1 || (ldx >= cols && ldy >= cols && (!resid || ldr >= cols))), "novic_dropout: rows, cols >= 0, leading dimensions >= cols");
	NOVIC_CHECK(cols == 0 || rows <= INT64_MAX / 8 / cols, "novic_dropout: too many elements");
	if (rows == 0 || cols == 0) return 0;
	NOVIC_CHECK(x && y, "novic_dropout: null pointer");
	const long long bx = type_bytes(x_type), by = type_bytes(y_type);
	NOVIC_APART("novic_dropout", NOVIC_SPANS({y, rows, cols * by, ldy * by}), NOVIC_SPANS({step, 1, 8, 0}, {x_type == y_type ? nullptr : x, rows, cols * bx, ldx * bx}),
	            NOVIC_SPANS({x_type == y_type ? x : nullptr, rows, cols * bx, ldx * bx}, {resid, rows, cols * by, ldr * by}))
	Args g;
	g.x = x; g.y = y; g.resid = resid;
	g.ldx = ldx; g.ldy = ldy; g.ldr = ldr;
	g.rows = rows; g.cols = cols;
	g.step = (const long long*)step;
	g.thr = (uint32_t)(p * 65536.0 + 0.5);
	g.scale = g.thr >= 65536u ? 0.f : (float)(65536.0 / (double)(65536u - g.thr));
	g.seed_lo = (uint32_t)seed; g.seed_hi = (uint32_t)(seed >> 32);
	g.site = site;
	if (x_type == NOVIC_TYPE_F32) NOVIC_TYPE_SWITCH(y_type, YT, (launch<float, YT>(g, stream)))
	else if (y_type == NOVIC_TYPE_F32) NOVIC_TYPE_SWITCH(x_type, XT, (launch<XT, float>(g, stream)))
	else NOVIC_TYPE_SWITCH(x_type, XT, (launch<XT, XT>(g, stream)))
	NOVIC_LAUNCH_CHECK();
	return 0;
}
