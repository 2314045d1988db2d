// Row access shared by the operators of decoder fine-tuning (layernorm_stats.hip, dropout.hip, token_loss.hip): a row of ANY width, at any element-aligned address, moved in
// whole vectors.  Lane `lane` of a row's team owns the chunks that start at e0 = (c * lanes + lane) * CH; the chunk that would leave the row is moved back to end with it
// (es = min(e0, E - CH)), so that every load is one full vector inside the row, without a branch.  Elements below e0 are then a neighbour's: they count in no sum and are not
// stored (an output may be one of the inputs).  gfx950 takes vector accesses at any address that its elements may have.
#pragma once
#include "common.hpp"

// N elements as they lie in memory: 16-bit ones two to a register (an array of them would be spread over a register each)
template <typename T, int N>
struct RawVec {
	static constexpr int WORDS = (int)sizeof(T) * N / 4;
	uint32_t w[WORDS];
	__device__ __forceinline__ float get(int i) const {
		if constexpr (sizeof(T) == 4) {
			return __uint_as_float(w[i]);
		} else if constexpr (__is_same(T, bf16)) {
			return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
		} else {
			return (float)__builtin_bit_cast(T, (unsigned short)(i & 1 ? w[i / 2] >> 16 : w[i / 2]));
		}
	}
	__device__ __forceinline__ void put(const float (&f)[N]) {
		if constexpr (sizeof(T) == 4) {
#pragma unroll
			for (int i = 0; i < N; ++i) w[i] = __float_as_uint(f[i]);
		} else {
			typedef T pair __attribute__((ext_vector_type(2)));
#pragma unroll
			for (int i = 0; i < N; i += 2) {
				const pair h = {(T)f[i], (T)f[i + 1]};
				__builtin_memcpy(&w[i / 2], &h, 4);
			}
		}
	}
};
template <typename T>
struct RawVec<T, 1> {
	T t;
	__device__ __forceinline__ float get(int) const { return (float)t; }
	__device__ __forceinline__ void put(const float (&f)[1]) { t = (T)f[0]; }
};
template <typename T, int N>
__device__ __forceinline__ RawVec<T, N> load_vec(const T* p) {
	RawVec<T, N> r;
	__builtin_memcpy(&r, p, sizeof(r));
	return r;
}
// the same, for what the kernel reads once: the caches need not keep it
template <typename T, int N>
__device__ __forceinline__ RawVec<T, N> load_once(const T* p) {
	RawVec<T, N> r;
	if constexpr (sizeof(r) % 8 == 0) {
		constexpr int W = sizeof(r) % 16 == 0 ? 4 : 2;
		typedef uint32_t words __attribute__((ext_vector_type(W), aligned(2), may_alias));
#pragma unroll
		for (int i = 0; i < RawVec<T, N>::WORDS; i += W) {
			const words q = __builtin_nontemporal_load((const words*)((const uint32_t*)p + i));
#pragma unroll
			for (int k = 0; k < W; ++k) r.w[i + k] = q[k];
		}
	} else {
		__builtin_memcpy(&r, p, sizeof(r));
	}
	return r;
}
// element e of a row: the offset is 32 bits, so that a row that is the same for the wave keeps its address in scalar registers
template <typename T>
__device__ __forceinline__ T* elem(T* row, int e) {
	return (T*)((char*)row + (uint32_t)e * (uint32_t)sizeof(T));
}
template <typename T>
__device__ __forceinline__ const T* elem(const T* row, int e) {
	return (const T*)((const char*)row + (uint32_t)e * (uint32_t)sizeof(T));
}
// (The vectors of words may stand for elements of any type: an output may be an input, and no load may pass a store that changes what it reads.)
// STREAM: past the caches (an output larger than they are, which nobody finds there again, leaves them to the inputs)
template <bool STREAM, typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[N]) {
	RawVec<T, N> r;
	r.put(f);
	if constexpr (STREAM && sizeof(r) % 16 == 0) {
		typedef uint32_t quad __attribute__((ext_vector_type(4), aligned(2), may_alias));
#pragma unroll
		for (int i = 0; i < (int)sizeof(r) / 16; ++i) {
			const quad q = {r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]};
			__builtin_nontemporal_store(q, (quad*)p + i);
		}
	} else {
		__builtin_memcpy(p, &r, sizeof(r));
	}
}
// The same values, out of the compiler's sight: what is computed from them again is not kept in registers over the code between.
template <typename T, int N>
__device__ __forceinline__ void forget(RawVec<T, N>& r) {
	if constexpr (N > 1) {
#pragma unroll
		for (int i = 0; i < RawVec<T, N>::WORDS; ++i) asm volatile("" : "+v"(r.w[i]));
	}
}
// the elements e0 .. of a chunk that was loaded at es <= e0, at row p
template <bool STREAM, typename T, int N>
__device__ __forceinline__ void store_own(T* p, int es, int e0, const float (&f)[N]) {
	if (es == e0) {
		store_vec<STREAM>(elem(p, es), f);
	} else {
#pragma unroll
		for (int i = 1; i < N; ++i)
			if (es + i >= e0) *elem(p, es + i) = (T)f[i];
	}
}

// sum over a team of LANES consecutive lanes (a power of two up to 64), everyone gets it
template <int LANES>
__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
	for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
	return v;
}
template <int LANES>
__device__ __forceinline__ float team_max(float v) {
#pragma unroll
	for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
	return v;
}

// element types of the C ABI (NOVIC_TYPE_*): calls F with a value of the C++ type
#define NOVIC_TYPE_SWITCH(type, T, CALL)                             \
	switch (type) {                                                  \
		case NOVIC_TYPE_F32: { typedef float T; CALL; break; }       \
		case NOVIC_TYPE_BF16: { typedef bf16 T; CALL; break; }       \
		default: { typedef f16 T; CALL; break; }                     \
	}
inline long long type_bytes(int type) { return type == NOVIC_TYPE_F32 ? 4 : 2; }

// ---- host side: an output that shares memory with another tensor of its call -----------------------------------------------------------------------------------------
struct Span {  // rows of `width` bytes, `ld` bytes apart; a null pointer is no tensor
	const void* p;
	long long rows, width, ld;
};
inline bool spans_meet(const Span& a, const Span& b) {
	if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
	const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
	const uintptr_t a1 = a0 + (uintptr_t)((a.rows - 1) * a.ld + a.width), b1 = b0 + (uintptr_t)((b.rows - 1) * b.ld + b.width);
	if (a0 >= b1 || b0 >= a1) return false;
	if (a.rows > 1 && b.rows > 1 && a.ld == b.ld) {  // column windows of one buffer that do not touch
		const long long shift = b0 >= a0 ? (long long)((b0 - a0) % (uintptr_t)a.ld) : (a.ld - (long long)((a0 - b0) % (uintptr_t)a.ld)) % a.ld;
		if (shift >= a.width && shift + b.width <= a.ld) return false;
	}
	return true;
}
inline bool same_span(const Span& a, const Span& b) { return a.p == b.p && a.rows == b.rows && a.width == b.width && (a.ld == b.ld || a.rows == 1); }
// `first`, an output, may be one of `may_be`; nothing else that is written may share memory with anything
inline bool spans_clash(const Span* outs, int n_out, const Span* ins, int n_in, const Span* may_be, int n_may) {
	for (int i = 0; i < n_out; ++i) {
		for (int j = 0; j < i; ++j)
			if (spans_meet(outs[i], outs[j])) return true;
		for (int j = 0; j < n_in; ++j)
			if (spans_meet(outs[i], ins[j])) return true;
		for (int j = 0; j < n_may; ++j)
			if (spans_meet(outs[i], may_be[j]) && !(i == 0 && same_span(outs[0], may_be[j]))) return true;
	}
	return false;
}
#define NOVIC_APART(what, OUTS, INS, MAY_BE)                                                                                        \
	{                                                                                                                               \
		const Span outs_[] = OUTS, ins_[] = INS, may_[] = MAY_BE;                                                                     \
		NOVIC_CHECK(!spans_clash(outs_, (int)(sizeof(outs_) / sizeof(Span)), ins_, (int)(sizeof(ins_) / sizeof(Span)), may_, (int)(sizeof(may_) / sizeof(Span))), \
		            what ": an output overlaps another tensor of the call");                                                            \
	}
#define NOVIC_SPANS(...) {__VA_ARGS__}
