/*
 * ndbhip_int8.hip — the 8-bit half of libndbhip.so: rows quantised to signed bytes with one scale each, the int8
 * matrix product of queries with a table of such rows, penalties / biases / masks over a matrix of scores, and the k
 * best rows of a table for every query.  Host entry points of include/ndbhip.h ("8-bit tables and scores").
 * Written for wave64 / CDNA4 (gfx950) only.
 *
 * Layout.  A table (and a batch of queries while a call runs) is kept in blocks of 32 rows; inside a block the
 * dimensions go in slices of 16: unit (row r, slice t) = 16 bytes at t * 512 + (r % 32) * 16.  Two neighbouring slices
 * are 1 KiB, and lane l of a wave reading 16 bytes at 16 l holds exactly what v_mfma_i32_32x32x32_i8 takes from lane l
 * as the A (or B) operand: row l % 32, bytes 16 (l / 32) .. + 15 of the 32.  So an operand is one contiguous KiB, from
 * memory or from LDS, with no shuffle and no bank conflict, and a block is one contiguous stream.  Dimensions are padded
 * with zeros to a multiple of 64, rows to a multiple of 256; a padding row's scale is NaN, which no search returns.
 */
#include "ndbhip_internal.h"
#include <hip/hip_fp16.h>
#include <hip/hip_bf16.h>
#include <mutex>
#include <new>

typedef int i8_v4i __attribute__((ext_vector_type(4)));
typedef int i8_v16i __attribute__((ext_vector_type(16)));

#define I8_ROW_PAD	256u		/* rows of a table are laid out in multiples of this (the widest tile) */
#define I8_DIM_PAD	64u
/* a row whose largest magnitude is below this is a row of zeros: 127 / top must stay finite */
#define I8_TINY		0x1p-100f
#define I8_NINF		(-__builtin_inff())

__host__ __device__ __forceinline__ uint32_t
i8_up(uint32_t v, uint32_t to)
{
	return (v + to - 1) / to * to;
}

/* ================================================================== */
/* element types                                                       */
/* ================================================================== */

template <class T> struct I8Elem;
template <> struct I8Elem<float>
{
	static __device__ __forceinline__ float load(float v) { return v; }
	static __device__ __forceinline__ float store(float v) { return v; }
};
template <> struct I8Elem<__half>
{
	static __device__ __forceinline__ float load(__half v) { return __half2float(v); }
	static __device__ __forceinline__ __half store(float v)
	{
		/* (left to itself the compiler folds a product and this into one mixed instruction that skips the rounding to fp32) */
		asm("" : "+v"(v));
		return __float2half_rn(v);
	}
};
template <> struct I8Elem<__hip_bfloat16>
{
	static __device__ __forceinline__ float load(__hip_bfloat16 v) { return __bfloat162float(v); }
	static __device__ __forceinline__ __hip_bfloat16 store(float v) { return __float2bfloat16(v); }
};

/* N neighbouring elements in one access.  Global memory takes any alignment (an odd number of halves a row costs nothing
 * but the lines that straddle), so there is one path for all strides. */
template <class T, int N> struct alignas(sizeof(T) * N) I8Vec
{
	T			v[N];
};
template <class T, int N>
__device__ __forceinline__ I8Vec<T, N>
i8_get(const void *p)
{
	I8Vec<T, N> v;

	__builtin_memcpy(&v, p, sizeof(v));
	return v;
}
template <class T, int N>
__device__ __forceinline__ void
i8_put(void *p, const I8Vec<T, N> &v)
{
	__builtin_memcpy(p, &v, sizeof(v));
}

/* ================================================================== */
/* quantise / dequantise                                               */
/* ================================================================== */

/*
 * byte = the integer nearest to x * inv, inv = RN(127 / top), halves to even.  One fused multiply-add onto 1.5 * 2^23
 * rounds the EXACT product to an integer once — RN(x * inv) first and rounding that would move products just beside a
 * half onto it — and leaves the integer in the low mantissa bits, whose low byte is the signed byte.
 */
__device__ __forceinline__ uint32_t
i8_byte(float x, float inv)
{
	return __float_as_uint(__builtin_fmaf(x, inv, 12582912.0f)) & 255u;
}

/*
 * L lanes (a power of two) hold a row, 64 / L rows a wave; a lane takes VEC neighbouring elements (16 bytes of input)
 * at a time.  The row's largest magnitude is an integer maximum over the magnitude bits, in which NaN and infinity are
 * largest and so cannot be lost.  Rows of up to CH * L * VEC elements stay in registers between the two passes; longer
 * ones are read again (from L2).  Short rows of a large matrix: R of them a lane at once, so that as much is under way as for
 * long ones (300 M elements in rows of 128: fp32 4.5 -> 5.8 TB/s, fp16 3.9 -> 5.7).  BLOCKED: bytes go to the block layout (rows from nrows on: zeros, scale NaN), else
 * to rows of `cstride` bytes.  Bound by HBM: e bytes read and one written per element (1M x 768 fp32 to rows: 702 us, 5.5
 * TB/s; to blocks, where 16 bytes of a row lie together: 975 us, 3.9 TB/s).
 */
template <class T, bool BLOCKED, int CH, int R>
__global__ __launch_bounds__(256) void
k_i8_quantize(const T *__restrict__ x, int64_t nrows, int64_t nrows_out, int dim, int64_t xstride, int lanes_log2,
			  unsigned char *__restrict__ codes, int64_t cstride, uint32_t kp, float *__restrict__ scales)
{
	constexpr int VEC = 16 / sizeof(T);
	const int	L = 1 << lanes_log2, per = 256 >> lanes_log2;
	const int	lane = threadIdx.x & (L - 1);
	const int64_t row0 = (int64_t) blockIdx.x * (per * R) + (threadIdx.x >> lanes_log2);
	const int	step = L * VEC;

	/* rows of bytes: the elements behind the last whole VEC are taken with those before them, which two lanes then write alike */
	auto		whole = [&](int e) -> int { return BLOCKED || dim < VEC || e >= dim ? e : min(e, dim - VEC); };
	auto		load = [&](int64_t row, int e0, float (&f)[VEC]) {
		const bool	real = row < nrows;
		const T    *p = x + (real ? row : 0) * xstride;
		const int	e = whole(e0);

		if (real && e + VEC <= dim)
		{
			const I8Vec<T, VEC> v = i8_get<T, VEC>(p + e);

#pragma unroll
			for (int i = 0; i < VEC; i++)
				f[i] = I8Elem<T>::load(v.v[i]);
		}
		else
#pragma unroll
			for (int i = 0; i < VEC; i++)
				f[i] = real && e + i < dim ? I8Elem<T>::load(p[e + i]) : 0.0f;
	};
	const bool	held = R > 1 || CH * step >= dim;
	float		reg[R][CH][VEC];

	if (held)
#pragma unroll
		for (int r = 0; r < R; r++)
#pragma unroll
			for (int c = 0; c < CH; c++)
				load(row0 + r * per, c * step + lane * VEC, reg[r][c]);
#pragma unroll
	for (int r = 0; r < R; r++)
	{
		const int64_t row = row0 + r * per;
		const bool	real = row < nrows;
		uint32_t	top = 0;

		if (held)
		{
#pragma unroll
			for (int c = 0; c < CH; c++)
#pragma unroll
				for (int i = 0; i < VEC; i++)
					top = max(top, __float_as_uint(reg[r][c][i]) & 0x7FFFFFFFu);
		}
		else
			for (int e = lane * VEC; e < dim; e += step)
			{
				load(row, e, reg[r][0]);
#pragma unroll
				for (int i = 0; i < VEC; i++)
					top = max(top, __float_as_uint(reg[r][0][i]) & 0x7FFFFFFFu);
			}
		for (int off = L >> 1; off > 0; off >>= 1)
			top = max(top, (uint32_t) __shfl_xor((int) top, off, 64));

		const float ftop = __uint_as_float(top);
		const bool	finite = top < 0x7F800000u;
		const bool	live = finite && ftop >= I8_TINY;
		const float inv = live ? 127.0f / ftop : 0.0f;

		if (row >= nrows_out)
			continue;			/* (a row's lanes together) */
		if (lane == 0)
			scales[row] = !real || !finite ? __builtin_nanf("") : live ? ftop / 127.0f : 0.0f;

		unsigned char *out = BLOCKED ? codes + (size_t) (row >> 5) * 32u * kp + (row & 31) * 16u : codes + row * cstride;
		auto		put = [&](int e0, const float (&f)[VEC]) {
			const int	e = whole(e0);
			I8Vec<uint32_t, VEC / 4> w;

#pragma unroll
			for (int i = 0; i < VEC / 4; i++)
				w.v[i] = live ? i8_byte(f[4 * i], inv) | i8_byte(f[4 * i + 1], inv) << 8 | i8_byte(f[4 * i + 2], inv) << 16 |
					i8_byte(f[4 * i + 3], inv) << 24 : 0u;
			if (BLOCKED)
				*(I8Vec<uint32_t, VEC / 4> *) (out + (size_t) (e >> 4) * 512u + (e & 15)) = w;
			else if (e + VEC <= dim)
				i8_put(out + e, w);
			else
#pragma unroll
				for (int i = 0; i < VEC; i++)
					if (e + i < dim)
						out[e + i] = (unsigned char) (w.v[i / 4] >> (8 * (i % 4)));
		};
		const int	end = BLOCKED ? (int) kp : dim;

		if (held)
		{
#pragma unroll
			for (int c = 0; c < CH; c++)
				if (c * step + lane * VEC < end)
					put(c * step + lane * VEC, reg[r][c]);
			if (BLOCKED)			/* padding dimensions beyond the registers' reach */
				for (int e = CH * step + lane * VEC; e < end; e += step)
				{
					load(row, e, reg[r][0]);
					put(e, reg[r][0]);
				}
		}
		else
			for (int e = lane * VEC; e < end; e += step)
			{
				load(row, e, reg[r][0]);
				put(e, reg[r][0]);
			}
	}
}

/*
 * byte * scale in fp32, rounded once more where the output has 16 bits; a lane takes the elements of a 16-byte store at a time,
 * CH loads of each of R rows ahead (R > 1: rows of no more than those).  TAIL: rows that are not whole stores (1M x 300 fp16 340 -> 158
 * us; rows that are lose up to 7 % by it).  Bound by HBM (1M x 768 to fp32: 684 us, 5.6 TB/s).
 */
template <class T, bool TAIL, int CH, int R>
__global__ __launch_bounds__(256) void
k_i8_dequantize(const int8_t *__restrict__ codes, int64_t cstride, const float *__restrict__ scales, int64_t nrows, int dim,
				int lanes_log2, T *__restrict__ out, int64_t ostride)
{
	constexpr int VEC = 16 / sizeof(T), W = VEC / 4;
	const int	L = 1 << lanes_log2, per = 256 >> lanes_log2;
	const int	lane = threadIdx.x & (L - 1);
	const int64_t row0 = (int64_t) blockIdx.x * (per * R) + (threadIdx.x >> lanes_log2);

	/* (as above: the end of a row with what is before it) */
	auto		whole = [&](int e) -> int { return !TAIL || dim < VEC || e >= dim ? e : min(e, dim - VEC); };

	for (int e0 = lane * VEC; e0 < dim; e0 += VEC * L * CH)
	{
		I8Vec<uint32_t, W> w[R][CH];
		float		s[R];

#pragma unroll
		for (int r = 0; r < R; r++)
		{
			const int64_t row = min(row0 + r * per, nrows - 1);		/* (behind the last row: that one again, not written) */
			const int8_t *c = codes + row * cstride;

			s[r] = scales[row];
#pragma unroll
			for (int u = 0; u < CH; u++)
			{
				const int	e = whole(e0 + u * VEC * L);

				if (e + VEC <= dim)
					w[r][u] = i8_get<uint32_t, W>(c + e);
				else
#pragma unroll
					for (int j = 0; j < W; j++)
					{
						w[r][u].v[j] = 0;
#pragma unroll
						for (int i = 0; i < 4; i++)
							w[r][u].v[j] |= e + 4 * j + i < dim ? (uint32_t) (uint8_t) c[e + 4 * j + i] << (8 * i) : 0u;
					}
			}
		}
#pragma unroll
		for (int r = 0; r < R; r++)
		{
			if (row0 + r * per >= nrows)
				break;
			T		   *o = out + (row0 + r * per) * ostride;

#pragma unroll
			for (int u = 0; u < CH; u++)
			{
				const int	e = whole(e0 + u * VEC * L);
				I8Vec<T, VEC> v;

#pragma unroll
				for (int i = 0; i < VEC; i++)
					v.v[i] = I8Elem<T>::store((float) (int8_t) (w[r][u].v[i / 4] >> (8 * (i % 4))) * s[r]);
				if (e + VEC <= dim)
					i8_put(o + e, v);
				else
#pragma unroll
					for (int i = 0; i < VEC; i++)
						if (e + i < dim)
							o[e + i] = v.v[i];
			}
		}
	}
}

/* rows of bytes <-> the block layout, 16 bytes a thread (neighbouring threads: neighbouring slices of a row) */
template <bool PACK>
__global__ __launch_bounds__(256) void
k_i8_blocks(const unsigned char *__restrict__ src, unsigned char *__restrict__ dst, int64_t stride, int64_t nrows, int64_t nrows_out,
			int dim, uint32_t kp, const float *__restrict__ sin, float *__restrict__ sout)
{
	const uint32_t slices = kp / 16;
	const uint64_t unit = (uint64_t) blockIdx.x * 256 + threadIdx.x;
	const int64_t row = unit / slices;
	const int	e = (int) (unit - (uint64_t) row * slices) * 16;

	if (row >= nrows_out)
		return;
	const size_t blk = (size_t) (row >> 5) * 32u * kp + (row & 31) * 16u + (size_t) (e >> 4) * 512u;
	I8Vec<unsigned char, 16> u;

	if (PACK)
	{
		const unsigned char *s = src + row * stride + e;

		if (row < nrows && e + 16 <= dim)
			u = i8_get<unsigned char, 16>(s);
		else
#pragma unroll
			for (int i = 0; i < 16; i++)
				u.v[i] = row < nrows && e + i < dim ? s[i] : 0;
		*(I8Vec<unsigned char, 16> *) (dst + blk) = u;
	}
	else
	{
		unsigned char *d = dst + row * stride + e;

		u = *(const I8Vec<unsigned char, 16> *) (src + blk);
		if (e + 16 <= dim)
			i8_put(d, u);
		else
#pragma unroll
			for (int i = 0; i < 16; i++)
				if (e + i < dim)
					d[i] = u.v[i];
	}
	if (e == 0)
		sout[row] = row < nrows ? sin[row] : __builtin_nanf("");
}

/* ================================================================== */
/* the product                                                         */
/* ================================================================== */

/* what becomes of a 32 x 32 block of sums: written as scores, or reduced to each query's largest of the 32 rows */
struct I8Out
{
	const float *rscale;		/* [rows padded] */
	const float *qscale;		/* [queries padded to 32] */
	const float *bias;			/* [n] or NULL */
	const uint32_t *mask;		/* bit i of word i / 32, or NULL */
	int64_t		mask_stride;	/* words from one query to the next; 0 = one mask for all */
	void	   *out;			/* scores */
	int64_t		ostride;
	float	   *gmax;			/* [nq][ngp]: the largest score of each block of 32 rows that takes part, -inf if none */
	float	   *qmax;			/* [nq][ngp / 4]: the largest of four blocks' */
	uint32_t	ngp;			/* a multiple of 8; behind the last block of rows: not read */
	uint32_t	n;
	uint32_t	nq;
};

/* RN(RN(RN(dot) * row scale) * query scale) (+ bias): the definition's own roundings, so that equal scores are equal */
__device__ __forceinline__ float
i8_score(int dot, float rs, float qs)
{
	return ((float) dot * rs) * qs;
}

/* a score or two; PAST: past the caches */
template <bool PAST, class V>
__device__ __forceinline__ void
i8_store(void *p, const V &v)
{
	if constexpr (sizeof(V) == 4)
	{
		typedef uint32_t word __attribute__((aligned(2)));
		uint32_t	w;

		__builtin_memcpy(&w, &v, 4);
		if (PAST)
			__builtin_nontemporal_store(w, (word *) p);
		else
			*(word *) p = w;
	}
	else
	{
		uint16_t	w;

		__builtin_memcpy(&w, &v, 2);
		if (PAST)
			__builtin_nontemporal_store(w, (uint16_t *) p);
		else
			*(uint16_t *) p = w;
	}
}

/*
 * Writes the block of sums of row block rb and the query block that starts at query q0.  The matrix instruction had the
 * queries as its first operand: lane l has row l % 32 and, in register 4 g + j, query 8 g + 4 (l / 32) + j, so that a store
 * covers 32 neighbouring scores of each of two queries, whatever the matrix's alignment.  rs, bias: of the lane's row;
 * qs: the block's 32 query scales, in LDS.
 */
template <bool BIAS, bool PAST, class T>
__device__ __forceinline__ void
i8_write_scores(const I8Out &o, float rs, float bias, const float *qs, uint32_t rb, uint32_t q0, const i8_v16i &acc)
{
	const int	lane = threadIdx.x & 63;
	const uint32_t r = rb * 32 + (lane & 31), qh = q0 + 4 * (lane >> 5);
	T		   *out = (T *) o.out + (int64_t) qh * o.ostride + r;
	float		s[16];

#pragma unroll
	for (int g4 = 0; g4 < 4; g4++)
	{
		const float4 q4 = *(const float4 *) (qs + 8 * g4 + 4 * (lane >> 5));
		const float qv[4] = {q4.x, q4.y, q4.z, q4.w};

#pragma unroll
		for (int j = 0; j < 4; j++)
		{
			s[4 * g4 + j] = i8_score(acc[4 * g4 + j], rs, qv[j]);
			if (BIAS)
				s[4 * g4 + j] = s[4 * g4 + j] + bias;
		}
	}
	if constexpr (sizeof(T) == 2)
		if (q0 + 32 <= o.nq && rb * 32 + 32 <= o.n)
		{
			/* 16 bits: two lanes trade a score, so that each stores two neighbouring ones of one query */
			const bool	odd = lane & 1;
			T		   *pair = out + (odd ? o.ostride - 1 : 0);

#pragma unroll
			for (int i = 0; i < 16; i += 2)
			{
				const float got = __uint_as_float((uint32_t) __builtin_amdgcn_mov_dpp((int) __float_as_uint(odd ? s[i] : s[i + 1]), 0xB1, 0xF, 0xF, true));
				I8Vec<T, 2> v;

				v.v[0] = I8Elem<T>::store(odd ? got : s[i]);
				v.v[1] = I8Elem<T>::store(odd ? s[i + 1] : got);
				i8_store<PAST>(pair + (int64_t) (8 * (i / 4) + i % 4) * o.ostride, v);
			}
			return;
		}
	if (r >= o.n)
		return;
#pragma unroll
	for (int i = 0; i < 16; i++)
		if (q0 + 32 <= o.nq || qh + 8 * (i / 4) + i % 4 < o.nq)
		{
			const I8Vec<T, 1> v = {{I8Elem<T>::store(s[i])}};

			i8_store<PAST>(out + (int64_t) (8 * (i / 4) + i % 4) * o.ostride, v);
		}
}

/*
 * The largest score that takes part among the 32 rows of a block, for the lane's query (both halves of the wave hold it).
 * The rows were the matrix instruction's first operand: lane l has query l % 32 and, in register 4 g + j, row 8 g + 4 (l / 32) + j.
 * rs, bias: the block's 32 row scales and biases (in LDS).  fmaxf drops NaN: rows of NaN scores, padding rows among them, never take
 * part.  A product with a positive finite query scale rises with its other factor and so does its rounding, hence without
 * a bias RN(t * qs) is taken of the largest t only.
 */
template <bool BIAS, bool MASK>
__device__ __forceinline__ float
i8_block_max(const float *rs, const float *bias, uint32_t bits, float qs, const i8_v16i &acc)
{
	const int	h = (threadIdx.x & 63) >> 5;
	const bool	rises = qs > 0.0f && qs < __builtin_inff();
	float		m = I8_NINF;

	if (!BIAS && __all(rises))
	{
#pragma unroll
		for (int g4 = 0; g4 < 4; g4++)
		{
			const float4 r4 = *(const float4 *) (rs + 8 * g4 + 4 * h);
			const float rv[4] = {r4.x, r4.y, r4.z, r4.w};

#pragma unroll
			for (int j = 0; j < 4; j++)
			{
				float		t = (float) acc[4 * g4 + j] * rv[j];

				if (MASK)
				{
					const uint32_t in = (uint32_t) __builtin_amdgcn_sbfe((int) (bits >> (4 * h)), 8 * g4 + j, 1);

					t = __uint_as_float((in & __float_as_uint(t)) | (~in & 0xFF800000u));
				}
				m = fmaxf(m, t);
			}
		}
		m = m > I8_NINF ? m * qs : I8_NINF;
	}
	else
#pragma unroll
		for (int g4 = 0; g4 < 4; g4++)
		{
			const float4 r4 = *(const float4 *) (rs + 8 * g4 + 4 * h);
			const float rv[4] = {r4.x, r4.y, r4.z, r4.w};
			const float4 b4 = BIAS ? *(const float4 *) (bias + 8 * g4 + 4 * h) : make_float4(0, 0, 0, 0);
			const float bv[4] = {b4.x, b4.y, b4.z, b4.w};

#pragma unroll
			for (int j = 0; j < 4; j++)
			{
				float		t = i8_score(acc[4 * g4 + j], rv[j], qs);

				if (BIAS)
					t = t + bv[j];
				if (MASK)
				{
					const uint32_t in = (uint32_t) __builtin_amdgcn_sbfe((int) (bits >> (4 * h)), 8 * g4 + j, 1);

					t = __uint_as_float((in & __float_as_uint(t)) | (~in & 0xFF800000u));
				}
				m = fmaxf(m, t);
			}
		}
	return fmaxf(m, __shfl_xor(m, 32, 64));
}

__device__ __forceinline__ uint32_t
i8_mask_word(const I8Out &o, uint32_t rb, uint32_t q)
{
	return q < o.nq && rb * 32 < o.n ? o.mask[(int64_t) q * o.mask_stride + rb] : 0u;
}

/* what an instance of the product kernels does with its sums */
template <int MODE_, bool BIAS_, bool MASK_, class T_> struct I8Kind
{
	static constexpr int MODE = MODE_;		/* 0 writes scores, 1 leaves maxima, 2 writes scores past the caches (tiles only) */
	static constexpr bool BIAS = BIAS_, MASK = MASK_;
	typedef T_	T;
};

/*
 * Few queries: a wave multiplies RW blocks of 32 rows with TB blocks of 32 queries straight from memory, U steps of 32
 * dimensions requested at a time; the queries stay in the caches.  What the sums are combined with is requested first.
 * Bound by HBM: the table is read once for every TB * 32 queries (one query, 1M x 768: 125 us, 6.1 TB/s).
 */
template <int RW, int TB, class KIND>
__global__ __launch_bounds__(256) void
k_i8_stream(const unsigned char *__restrict__ rows, const unsigned char *__restrict__ queries, uint32_t kp, uint32_t nrb, I8Out o)
{
	constexpr int U = TB == 1 ? 8 : 4;
	__shared__ __attribute__((aligned(16))) float s_m[KIND::MODE == 1 ? TB * 32 : 1][4 * RW];
	__shared__ __attribute__((aligned(16))) float s_rs[4 * RW][32], s_bias[KIND::BIAS ? 4 * RW : 1][32];
	__shared__ __attribute__((aligned(16))) float s_qs[4][KIND::MODE != 1 ? TB * 32 : 1];
	const int	lane = threadIdx.x & 63;
	const int	wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const uint32_t qb0 = blockIdx.y * TB;
	const unsigned char *b = queries + (size_t) qb0 * 32u * kp + lane * 16;
	const unsigned char *a[RW];
	uint32_t	rb[RW];
	float		my_rs[RW], my_bias[RW], qs[TB];
	uint32_t	bits[RW][TB];
	i8_v16i		acc[RW][TB];

#pragma unroll
	for (int i = 0; i < RW; i++)
	{
		/* (waves behind the last block do it over) */
		rb[i] = min((blockIdx.x * 4 + wave) * RW + i, nrb - 1);
		a[i] = rows + (size_t) rb[i] * 32u * kp + lane * 16;

		const uint32_t row = rb[i] * 32 + (lane & 31);

		my_rs[i] = o.rscale[row];
		my_bias[i] = KIND::BIAS && row < o.n ? o.bias[row] : 0.0f;
	}
#pragma unroll
	for (int t = 0; t < TB; t++)
	{
		const uint32_t q = (qb0 + t) * 32 + (lane & 31);

		qs[t] = q < o.nq ? o.qscale[q] : 1.0f;
#pragma unroll
		for (int i = 0; i < RW; i++)
		{
			bits[i][t] = KIND::MASK ? i8_mask_word(o, rb[i], q) : 0u;
#pragma unroll
			for (int e = 0; e < 16; e++)
				acc[i][t][e] = 0;
		}
	}
	for (uint32_t k = 0; k < kp; k += 32 * U)
	{
		i8_v4i		av[U][RW], bv[U][TB];

		/* (a step behind the last one asks for that one again and is not multiplied) */
#pragma unroll
		for (int u = 0; u < U; u++)
#pragma unroll
			for (int i = 0; i < RW; i++)
				av[u][i] = *(const i8_v4i *) (a[i] + (size_t) min(k + u * 32, kp - 32) * 32);
#pragma unroll
		for (int u = 0; u < U; u++)
#pragma unroll
			for (int t = 0; t < TB; t++)
				bv[u][t] = *(const i8_v4i *) (b + (size_t) t * 32 * kp + (size_t) min(k + u * 32, kp - 32) * 32);
#pragma unroll
		for (int u = 0; u < U; u++)
			if (k + u * 32 < kp)
#pragma unroll
				for (int i = 0; i < RW; i++)
#pragma unroll
					for (int t = 0; t < TB; t++)
						acc[i][t] = KIND::MODE != 1 ? __builtin_amdgcn_mfma_i32_32x32x32_i8(bv[u][t], av[u][i], acc[i][t], 0, 0, 0) :
							__builtin_amdgcn_mfma_i32_32x32x32_i8(av[u][i], bv[u][t], acc[i][t], 0, 0, 0);
	}
	/* (a wave's own LDS: what it writes it reads in order) */
	if (lane < 32)
	{
#pragma unroll
		for (int i = 0; i < RW; i++)
		{
			s_rs[wave * RW + i][lane] = my_rs[i];
			if (KIND::BIAS)
				s_bias[wave * RW + i][lane] = my_bias[i];
		}
		if (KIND::MODE != 1)
#pragma unroll
			for (int t = 0; t < TB; t++)
				s_qs[wave][t * 32 + lane] = qs[t];
	}
	__builtin_amdgcn_wave_barrier();
#pragma unroll
	for (int t = 0; t < TB; t++)
#pragma unroll
		for (int i = 0; i < RW; i++)
			if (KIND::MODE != 1)
				i8_write_scores<KIND::BIAS, false, typename KIND::T>(o, my_rs[i], my_bias[i], s_qs[wave] + t * 32, rb[i],
																			   (qb0 + t) * 32, acc[i][t]);
			else
			{
				const float m = i8_block_max<KIND::BIAS, KIND::MASK>(s_rs[wave * RW + i], s_bias[KIND::BIAS ? wave * RW + i : 0], bits[i][t],
																	 qs[t], acc[i][t]);

				if (lane < 32)
					s_m[t * 32 + lane][wave * RW + i] = m;
			}
	if (KIND::MODE == 1)
	{
		__syncthreads();
		for (int e = threadIdx.x; e < TB * 32 * RW; e += 256)
		{
			const uint32_t q = qb0 * 32 + e / RW, quad = blockIdx.x * RW + e % RW;

			if (q < o.nq && quad * 4 < o.ngp)
			{
				const float4 m = *(const float4 *) &s_m[e / RW][e % RW * 4];

				*(float4 *) (o.gmax + (size_t) q * o.ngp + quad * 4) = m;
				o.qmax[(size_t) q * (o.ngp / 4) + quad] = fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w));
			}
		}
	}
}

/* ------------------------------------------------------------------ */

/* every request of this wave older than the newest N has landed */
template <int N>
__device__ __forceinline__ void
i8_wait_vm()
{
	static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit counter");
	asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}

/* lane i copies 16 (4) bytes at base + voff to LDS at la + 16 (4) i.  Inline asm: the compiler would put a wait for ALL
 * such copies in front of every LDS read of a ring it cannot tell apart, and M0, which only these copies use here, is
 * written right before each (the wait states cover M0 and a base that a vector instruction has just put into its scalar
 * registers).  M0 is named as written: the compiler keeps nothing in it from one instruction to another and so warns, but it
 * may share one setting of it between instructions, and must not across these.  Not a memory clobber: the barriers around the
 * ring are, and copies may move between reads. */
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void
i8_dma16(const void *base, uint32_t voff, uint32_t la)
{
	asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(la), "v"(voff), "s"(base) : "m0");
}
__device__ __forceinline__ void
i8_dma4(const void *base, uint32_t voff, uint32_t la)
{
	asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" :: "s"(la), "v"(voff), "s"(base) : "m0");
}

/* the same from 64 unrelated addresses */
__device__ __forceinline__ void
i8_dma4_at(const void *p, uint32_t la)
{
	asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, off" :: "s"(la), "v"(p) : "m0");
}
#pragma clang diagnostic pop

template <class T>
__device__ __forceinline__ T *
i8_uniform(T *p)
{
	const uint64_t v = (uint64_t) p;
	const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t) v), hi = __builtin_amdgcn_readfirstlane((uint32_t) (v >> 32));

	return (T *) (((uint64_t) hi << 32) | lo);
}

__device__ __forceinline__ uint32_t
i8_lds(const void *p)
{
	return (uint32_t) (uintptr_t) (__attribute__((address_space(3))) const unsigned char *) p;
}

/*
 * Many queries: a block of 2 x NWQ waves multiplies tiles of 256 rows x 64 NWQ queries, wave (wr, wq) of it 128 x 64 sums
 * in registers.  Both operands pass through LDS in stages of 64 dimensions (2 KiB a block of 32 rows
 * or queries, copied as they lie in memory; an LDS read is 16 bytes a lane without conflicts), a ring of NBUF.
 *
 * Two waves a SIMD do not hide each other's waits (those of a wide tile meet at the same barriers), so the stream is pipelined
 * by hand.  A stage is two halves of 32 dimensions (one matrix instruction deep): while one half is multiplied, the operands of
 * the next are read, also across the barrier that opens the next stage.  The ring runs into the next tile of the block, whose
 * first operands are in registers when the sums of this one are written out.
 *
 * Row scales, query scales, biases and mask words of a tile come through LDS the same way, with the copies of its first stage: a load
 * of the wave's own would have to wait for every copy requested before it (requests retire in order).
 *
 * Scores are the gap that is left: they count among the requests that the next stage waits for, and retire in order, so a
 * tile's 128 stores a wave (64 in 16 bits) are nearly all done before the next tile's first half stage ends.
 *
 * Bound by LDS and the matrix pipe together, and the clock they run at: a half stage moves 48 KiB out of LDS and 16 in, 512
 * cycles at 128 bytes each, and is 512 cycles of the pipe.  1024 x 1M x 768 to maxima 724 us (2.2 POP/s, the pipe busy 55 % of
 * the cycles; 690 on another box, and 570 there on zeros; 635 without the epilogue, 449 without the operands' LDS reads as well),
 * 1024 x 131072 x 1536 to fp32 scores 217, 77 x 50021 x 300 bf16 11.
 */
#define I8_TR 8					/* blocks of rows in a tile */
#define I8_NBUF 3
#define I8_SLOTS 4				/* tiles whose scales are in LDS: the ring is at most NBUF tiles ahead */

#define I8_WQ 2					/* blocks of queries a wave multiplies */

template <int NWQ> struct I8Tile
{
	static constexpr int NW = 2 * NWQ;
	static constexpr int QB = NWQ * I8_WQ;					/* blocks of queries in a tile */
	static constexpr int STAGE = (I8_TR + QB) * 2048;
	static constexpr int PER = 2 * (I8_TR + QB) / NW;		/* copies of 1 KiB a wave makes per stage */
};

template <int NWQ, class KIND>
__global__ __launch_bounds__(128 * NWQ, NWQ == 2 && (KIND::BIAS || KIND::MASK) ? 1 : 2) void
k_i8_tile(const unsigned char *__restrict__ rows, const unsigned char *__restrict__ queries, uint32_t kp, uint32_t nrt, uint32_t nqt, I8Out o)
{
	typedef I8Tile<NWQ> TILE;
	constexpr int QB = TILE::QB, PER = TILE::PER, WQ = I8_WQ;
	static_assert(WQ == 2, "a wave's queries are its lanes in the copies of mask words");
	__shared__ __attribute__((aligned(1024))) unsigned char ring[I8_NBUF * TILE::STAGE];
	__shared__ __attribute__((aligned(1024))) float s_rs[I8_SLOTS][256];
	__shared__ __attribute__((aligned(1024))) float s_qs[I8_SLOTS][256];
	__shared__ __attribute__((aligned(1024))) float s_bias[KIND::BIAS ? I8_SLOTS : 1][256];
	__shared__ __attribute__((aligned(1024))) uint32_t s_mask[KIND::MASK ? I8_SLOTS : 1][KIND::MASK ? TILE::NW : 1][4][64];
	const int	lane = threadIdx.x & 63;
	const int	wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int	wq = wave % NWQ, wr = wave / NWQ;
	/*
	 * Blocks go round the 8 XCDs.  An XCD takes every eighth row tile and of each all query tiles one after the other, dealt
	 * to its blocks in turn: its L2 holds the queries and sees each row tile once.
	 */
	const uint32_t xcd = blockIdx.x & 7, nslot = gridDim.x >> 3;
	const uint32_t mine = nrt > xcd ? (nrt - xcd + 7) / 8 * nqt : 0;
	const uint32_t blk = kp * 32;			/* bytes of a block */
	const uint32_t ns = kp / 64;
	const uint32_t ring_la = i8_lds(ring);
	const uint32_t first = blockIdx.x >> 3;

	if (first >= mine)
		return;
	const uint32_t dr = nslot / nqt, dq = nslot % nqt;		/* from a tile of this block to its next */
	auto		forward = [&](uint32_t &rt, uint32_t &qt) {
		rt += 8 * dr;
		qt += dq;
		if (qt >= nqt)
		{
			qt -= nqt;
			rt += 8;
		}
	};

	/* the copies' place in the stream of stages; behind the last tile they go over that one again, read by nobody */
	uint32_t	c_rt = first / nqt * 8 + xcd, c_qt = first % nqt, c_left = (mine - first + nslot - 1) / nslot, c_s = 0, c_slot = 0, c_buf = 0;
	const unsigned char *c_r = i8_uniform(rows + (size_t) c_rt * I8_TR * blk), *c_q = i8_uniform(queries + (size_t) c_qt * QB * blk);

	/* the first copies of a tile: its scales (and biases, the rows behind the last take the last one's) */
	auto		c_scales = [&]() {
		if (wave == 0)
			i8_dma16(i8_uniform(o.rscale + (size_t) c_rt * 256), lane * 16, i8_lds(s_rs) + c_slot * 1024);
		if (wave == 1)
			i8_dma16(i8_uniform(o.qscale + (size_t) c_qt * QB * 32), (lane & (QB * 8 - 1)) * 16, i8_lds(s_qs) + c_slot * 1024);
		if (KIND::BIAS && wave < 4)
			i8_dma4(i8_uniform(o.bias + (size_t) c_rt * 256), min(wave * 64u + lane, o.n - 1 - c_rt * 256) * 4,
					i8_lds(s_bias) + c_slot * 1024 + wave * 256);
		if (KIND::MASK)
		{
			/* the words of this wave's 64 queries, a lane each, for its four blocks of rows (the last query's and the last
			 * block's again behind them: padding rows never take part, and nobody asks for padding queries) */
			const uint32_t q = min((c_qt * QB + wq * WQ) * 32 + lane, o.nq - 1), nw = (o.n + 31) / 32;
			const uint32_t *m = o.mask + (int64_t) q * o.mask_stride;

#pragma unroll
			for (int i = 0; i < 4; i++)
				i8_dma4_at(m + min(c_rt * I8_TR + wr * 4 + i, nw - 1), i8_lds(s_mask) + ((c_slot * TILE::NW + wave) * 4 + i) * 256);
		}
	};
	auto		c_copy = [&](int i) {
		const int	c = wave * PER + i;			/* KiB c of the stage: block c / 2, half c % 2 */
		const bool	isq = c >= 2 * I8_TR;
		const uint32_t off = (uint32_t) ((isq ? c - 2 * I8_TR : c) >> 1) * blk + c_s * 2048u + (c & 1) * 1024u;

		i8_dma16(isq ? c_q : c_r, off + lane * 16, ring_la + c_buf * TILE::STAGE + c * 1024);
	};
	auto		c_next = [&]() {
		c_buf = c_buf + 1 == I8_NBUF ? 0 : c_buf + 1;
		if (++c_s == ns)
		{
			c_s = 0;
			c_slot = (c_slot + 1) & (I8_SLOTS - 1);
			if (--c_left > 0)
			{
				forward(c_rt, c_qt);
				c_r = i8_uniform(rows + (size_t) c_rt * I8_TR * blk);
				c_q = i8_uniform(queries + (size_t) c_qt * QB * blk);
			}
			else
				c_left = 1;
		}
	};

	i8_v4i		av[2][4], bv[2][WQ];
	i8_v16i		acc[4][WQ];
	const unsigned char *lane_ring = ring + lane * 16;
	auto		read = [&](uint32_t buf, int h) {
		const unsigned char *st = lane_ring + buf * TILE::STAGE + h * 1024;

#pragma unroll
		for (int t = 0; t < WQ; t++)
			bv[h][t] = *(const i8_v4i *) (st + (I8_TR + wq * WQ + t) * 2048);
#pragma unroll
		for (int i = 0; i < 4; i++)
			av[h][i] = *(const i8_v4i *) (st + (wr * 4 + i) * 2048);
	};

#pragma unroll
	for (int s = 0; s < I8_NBUF; s++)
	{
		if (c_s == 0)
			c_scales();
#pragma unroll
		for (int i = 0; i < PER; i++)
			c_copy(i);
		c_next();
	}
	i8_wait_vm<(I8_NBUF - 1) * PER>();
	asm volatile("s_barrier" ::: "memory");
	read(0, 0);

	uint32_t	buf = 0, slot = 0;
	auto		mul = [](const i8_v4i &r, const i8_v4i &q, const i8_v16i &c) -> i8_v16i {
		return KIND::MODE != 1 ? __builtin_amdgcn_mfma_i32_32x32x32_i8(q, r, c, 0, 0, 0) :
			__builtin_amdgcn_mfma_i32_32x32x32_i8(r, q, c, 0, 0, 0);
	};

	/*
	 * A stage, its first half's operands in registers.  FIRST: the tile's first stage, sums start from zero.  The next stage
	 * must have landed for every wave, and every wave must have read the last of this one, before the barrier in the middle;
	 * behind it this stage's place is filled again.
	 */
	auto		stage = [&](auto first_stage) {
		constexpr bool FIRST = decltype(first_stage)::value;
		const i8_v16i zero = {};

		read(buf, 1);
		__builtin_amdgcn_sched_barrier(0);
#pragma unroll
		for (int i = 0; i < 4; i++)
#pragma unroll
			for (int t = 0; t < WQ; t++)
				acc[i][t] = mul(av[0][i], bv[0][t], FIRST ? zero : acc[i][t]);
		__builtin_amdgcn_sched_barrier(0);
		i8_wait_vm<(I8_NBUF - 2) * PER>();
		asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
		buf = buf + 1 == I8_NBUF ? 0 : buf + 1;
		read(buf, 0);
		if (c_s == 0)
			c_scales();
		__builtin_amdgcn_sched_barrier(0);
#pragma unroll
		for (int i = 0; i < 4; i++)
#pragma unroll
			for (int t = 0; t < WQ; t++)
			{
				acc[i][t] = mul(av[1][i], bv[1][t], acc[i][t]);
				if (i * WQ + t < PER)
					c_copy(i * WQ + t);
				__builtin_amdgcn_sched_barrier(0);
			}
		c_next();
	};
	uint32_t	rt = first / nqt * 8 + xcd, qt = first % nqt;

	for (uint32_t left = (mine - first + nslot - 1) / nslot; left > 0; left--)
	{
		const uint32_t rb0 = rt * I8_TR + wr * 4, qb0 = qt * QB + wq * WQ;

		stage(std::true_type{});
		for (uint32_t s = 1; s < ns; s++)
			stage(std::false_type{});
#pragma unroll
		for (int t = 0; t < WQ; t++)
		{
			if (KIND::MODE != 1)
			{
#pragma unroll
				for (int i = 0; i < 4; i++)
					i8_write_scores<KIND::BIAS, KIND::MODE == 2, typename KIND::T>(o, s_rs[slot][(wr * 4 + i) * 32 + (lane & 31)],
																  s_bias[KIND::BIAS ? slot : 0][(wr * 4 + i) * 32 + (lane & 31)],
																  s_qs[slot] + (wq * WQ + t) * 32, rb0 + i, (qb0 + t) * 32, acc[i][t]);
			}
			else
			{
				const uint32_t q = (qb0 + t) * 32 + (lane & 31);
				const float qs = s_qs[slot][(wq * WQ + t) * 32 + (lane & 31)];
				float		m[4];

#pragma unroll
				for (int i = 0; i < 4; i++)
					m[i] = i8_block_max<KIND::BIAS, KIND::MASK>(s_rs[slot] + (wr * 4 + i) * 32,
																s_bias[KIND::BIAS ? slot : 0] + (wr * 4 + i) * 32,
																KIND::MASK ? s_mask[KIND::MASK ? slot : 0][KIND::MASK ? wave : 0][i][t * 32 + (lane & 31)] : 0u,
																q < o.nq ? qs : 1.0f, acc[i][t]);
				if (q < o.nq && lane < 32)
				{
					*(float4 *) (o.gmax + (size_t) q * o.ngp + rb0) = make_float4(m[0], m[1], m[2], m[3]);
					o.qmax[(size_t) q * (o.ngp / 4) + rb0 / 4] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
				}
			}
		}
		slot = (slot + 1) & (I8_SLOTS - 1);
		forward(rt, qt);
	}
	i8_wait_vm<0>();			/* (no copy may be on its way into LDS that is no longer this block's) */
}

/* ================================================================== */
/* the k best                                                          */
/* ================================================================== */

/*
 * Any k best rows lie in the k row blocks with the largest maxima (equal maxima: the lower block first): a row of
 * another block has k rows ahead of it, one in each of those blocks.  So the product leaves one number per (query, 32
 * rows) and one per (query, four such blocks); k quads are picked, of their blocks k, and only the rows of those are scored
 * again, one by one and with the same roundings.  The same holds at every step: the k-th of the maxima picked is a
 * floor under the k-th best of what lies below them, so that a step looks at little more than k candidates.
 *
 * What is selected is ordered by one 64-bit word, larger scores first and then lower ids; all of them differ.
 */
__device__ __forceinline__ uint64_t
i8_word(float v, uint32_t id)
{
	return (uint64_t) ndb_key_from_bits(__float_as_uint(-v)) << 32 | id;
}
__device__ __forceinline__ float
i8_word_score(uint64_t w)
{
	const uint32_t k = (uint32_t) (w >> 32);

	return -__uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k) + 0.0f;	/* (-0 and 0 are equal scores: 0) */
}

template <int NT, int CAP> struct I8Select
{
	uint64_t	list[CAP];
	uint32_t	hist[256], sh[16];
	float		top[NT];
	float		floor;
	uint32_t	cnt;
};

/* list[0 .. m) ascending; m <= CAP, a power of two.  Counting ranks beats the network's barriers for a few hundred words. */
template <int NT, int CAP>
__device__ void
i8_sort(I8Select<NT, CAP> &S, uint32_t m)
{
	if (m <= 512)
	{
		uint64_t	v[(512 + NT - 1) / NT];
		uint32_t	r[(512 + NT - 1) / NT];

#pragma unroll
		for (int e = 0; e < (512 + NT - 1) / NT; e++)
			if (threadIdx.x + e * NT < m)
			{
				v[e] = S.list[threadIdx.x + e * NT];
				r[e] = lds_rank_u64(S.list, m, v[e]);
			}
		__syncthreads();
#pragma unroll
		for (int e = 0; e < (512 + NT - 1) / NT; e++)
			if (threadIdx.x + e * NT < m)
				S.list[r[e]] = v[e];
		__syncthreads();
		return;
	}
	uint32_t	npad = 1024;

	while (npad < m)
		npad <<= 1;
	for (uint32_t i = m + threadIdx.x; i < npad; i += NT)
		S.list[i] = ~0ull;
	for (uint32_t size = 2; size <= npad; size <<= 1)
		for (uint32_t stride = size >> 1; stride > 0; stride >>= 1)
		{
			__syncthreads();
			for (uint32_t t = threadIdx.x; t < (npad >> 1); t += NT)
			{
				const uint32_t lo = 2 * t - (t & (stride - 1)), hi = lo + stride;
				const uint64_t x = S.list[lo], y = S.list[hi];

				if ((x > y) == ((lo & size) == 0))
				{
					S.list[lo] = y;
					S.list[hi] = x;
				}
			}
		}
	__syncthreads();
}

/*
 * The elements f(i, score, id) -> takes part, i = 0 .. n - 1, that reach `floor`, as words in S.list in no order; returns how
 * many.  At least min(k, valid) have to reach it.  Where more do than the list holds (many equal scores), the k best: the
 * k-th score is found by radix selection, and the k-th id among its equals.  Ends with a barrier.
 */
template <int NT, int CAP, class F>
__device__ uint32_t
i8_gather(I8Select<NT, CAP> &S, F f, uint32_t n, uint32_t k, float floor)
{
	if (threadIdx.x == 0)
		S.cnt = 0;
	__syncthreads();
	for (uint32_t i = threadIdx.x; i < n; i += NT)
	{
		float		v;
		uint32_t	id;

		if (f(i, v, id) && v >= floor)
		{
			const uint32_t at = atomicAdd(&S.cnt, 1u);

			if (at < CAP)
				S.list[at] = i8_word(v, id);
		}
	}
	__syncthreads();
	const uint32_t m = S.cnt;

	if (m <= CAP)
		return m;

	uint32_t	T, less, kk, eq, T2 = ~0u;

	block_radix_select([&](uint32_t i, uint32_t &bits) -> bool {
		float		v;
		uint32_t	id;
		const bool	ok = f(i, v, id);

		bits = __float_as_uint(-v);
		return ok;
	}, n, k, S.hist, S.sh, T, less, kk, eq);
	if (eq > kk - less)
	{
		uint32_t	l2, k2, e2;

		block_radix_select([&](uint32_t i, uint32_t &bits) -> bool {
			float		v;
			const bool	ok = f(i, v, bits);

			return ok && ndb_key_from_bits(__float_as_uint(-v)) == T;
		}, n, kk - less, S.hist, S.sh, T2, l2, k2, e2);
	}
	if (threadIdx.x == 0)
		S.cnt = 0;
	__syncthreads();
	for (uint32_t i = threadIdx.x; i < n; i += NT)
	{
		float		v;
		uint32_t	id;

		if (!f(i, v, id))
			continue;
		const uint32_t key = ndb_key_from_bits(__float_as_uint(-v));

		/* (ids are below 2^31: as keys of floats they keep their order) */
		if (key < T || (key == T && ndb_key_from_bits(id) <= T2))
			S.list[atomicAdd(&S.cnt, 1u)] = i8_word(v, id);
	}
	__syncthreads();
	return kk;
}

/* the min(k, valid) best of them in order; returns how many */
template <int NT, int CAP, class F>
__device__ uint32_t
i8_select(I8Select<NT, CAP> &S, F f, uint32_t n, uint32_t k, float floor)
{
	const uint32_t m = i8_gather(S, f, n, k, floor);

	i8_sort(S, m);
	return min(m, k);
}

/*
 * A floor under the k-th largest of top[0 .. groups), k <= groups <= 64 N, by one wave: the leading 20 bits of the
 * largest key that k of them reach (sign, exponent and 11 bits of the mantissa: within 2^-11 below the k-th itself).
 */
template <int N>
__device__ __forceinline__ float
i8_floor(const float *top, uint32_t groups, uint32_t k)
{
	const int	lane = threadIdx.x & 63;
	uint32_t	key[N], T = 0;

#pragma unroll
	for (int e = 0; e < N; e++)
	{
		const uint32_t i = e * 64 + lane;

		/* (larger scores: larger keys; nothing: 0, which no threshold but 0 admits) */
		key[e] = i < groups && top[i] > I8_NINF ? ndb_key_from_bits(__float_as_uint(top[i])) : 0u;
	}
	for (uint32_t bit = 0x80000000u; bit >= 0x1000u; bit >>= 1)
	{
		uint32_t	c = 0;

#pragma unroll
		for (int e = 0; e < N; e++)
			c += __popcll(__ballot(key[e] >= (T | bit)));
		if (c >= k)
			T |= bit;
	}
	if (T == 0)
		return I8_NINF;
	const float f = __uint_as_float((T & 0x80000000u) ? T ^ 0x80000000u : ~T);

	return f == f ? f : I8_NINF;	/* (between -infinity's key and the smallest number's lie those of NaN) */
}

/*
 * The k best blocks of 32 rows of a query, in S.list; returns how many there are.  The floor of every step: k of about 2k .. 4k
 * groups of threads have a quad that reaches it.
 */
template <int NT, int CAP>
__device__ uint32_t
i8_pick(I8Select<NT, CAP> &S, uint32_t (&quads)[CAP], const float *gm, const float *qm, uint32_t ng, uint32_t k)
{
	const uint32_t nquad = (ng + 3) / 4;
	const uint32_t span = min(nquad, (uint32_t) NT);
	float		t = I8_NINF;
	uint32_t	size = 64;			/* threads of a group, neighbours in a wave */

	while (size > 1 && span < 2 * k * size)
		size >>= 1;
	const uint32_t groups = (span + size - 1) / size;

	for (uint32_t i = threadIdx.x; i < nquad; i += 8 * NT)
	{
		float		v[8];

#pragma unroll
		for (int e = 0; e < 8; e++)
			v[e] = i + e * NT < nquad ? qm[i + e * NT] : I8_NINF;
#pragma unroll
		for (int e = 0; e < 8; e++)
			t = fmaxf(t, v[e]);
	}
	for (uint32_t off = 1; off < size; off <<= 1)
		t = fmaxf(t, __shfl_xor(t, off, 64));
	if (threadIdx.x % size == 0)
		S.top[threadIdx.x / size] = t;
	__syncthreads();
	if (threadIdx.x < 64)
	{
		const float f = k > groups ? I8_NINF : groups <= 64 ? i8_floor<1>(S.top, groups, k) : groups <= 256 ?
			i8_floor<4>(S.top, groups, k) : i8_floor<NT / 64>(S.top, groups, k);

		if (threadIdx.x == 0)
			S.floor = f;
	}
	__syncthreads();
	const float floor = S.floor;
	const uint32_t m = i8_gather(S, [&](uint32_t i, float &v, uint32_t &id) -> bool {
		v = qm[i];
		id = i;
		return v > I8_NINF;
	}, nquad, k, floor);

	for (uint32_t i = threadIdx.x; i < m; i += NT)
		quads[i] = (uint32_t) S.list[i];
	__syncthreads();
	return i8_select(S, [&](uint32_t i, float &v, uint32_t &id) -> bool {
		id = quads[i / 4] * 4 + i % 4;
		v = id < ng ? gm[id] : I8_NINF;
		return v > I8_NINF;
	}, m * 4, k, floor);
}

/*
 * Scoring picked blocks again.  A wave takes a part, up to 8 steps of 32 dimensions, of one block and asks for all of it at
 * once: the rows are anywhere in the table, so what counts is how many requests are under way.  A lane sums 16-byte pieces
 * of row l % 32 against the query's, the two halves of the wave are joined, and the parts of a block add up in LDS.
 */
#define I8_PART 8u
__device__ __forceinline__ int
i8_part_sum(const unsigned char *rows, const unsigned char *queries, uint32_t kp, uint32_t rb, uint32_t q, uint32_t part)
{
	const int	lane = threadIdx.x & 63;
	const uint32_t e0 = part * I8_PART * 32;
	const unsigned char *a = rows + (size_t) rb * 32u * kp + lane * 16;
	const unsigned char *b = queries + (size_t) (q >> 5) * 32u * kp + (q & 31) * 16 + (lane >> 5) * 512;
	i8_v4i		x[I8_PART], y[I8_PART];
	int			s = 0;

#pragma unroll
	for (uint32_t u = 0; u < I8_PART; u++)
		if (e0 + u * 32 < kp)
		{
			x[u] = *(const i8_v4i *) (a + (size_t) (e0 + u * 32) * 32);
			y[u] = *(const i8_v4i *) (b + (size_t) (e0 + u * 32) * 32);
		}
#pragma unroll
	for (uint32_t u = 0; u < I8_PART; u++)
		if (e0 + u * 32 < kp)
#pragma unroll
			for (int i = 0; i < 4; i++)
				s = __builtin_amdgcn_sdot4(x[u][i], y[u][i], s, false);
	return s + __shfl_xor(s, 32, 64);
}

/* what the sums of row i of block rb become a score with */
struct I8Row
{
	float		rs, bias;
	uint32_t	bits;
};
__device__ __forceinline__ I8Row
i8_row(const I8Out &o, uint32_t rb, uint32_t i, uint32_t q)
{
	const uint32_t r = rb * 32 + i;
	I8Row		w;

	w.rs = o.rscale[r];
	w.bias = o.bias && r < o.n ? o.bias[r] : 0.0f;
	w.bits = o.mask ? o.mask[(int64_t) q * o.mask_stride + rb] >> i : 1u;
	return w;
}
/* -inf for rows that take no part */
__device__ __forceinline__ float
i8_row_score(const I8Out &o, const I8Row &w, int dot, float qs)
{
	float		v = i8_score(dot, w.rs, qs);

	if (o.bias)
		v = v + w.bias;
	return v > I8_NINF && (w.bits & 1u) ? v : I8_NINF;
}

template <int NT>
__device__ __forceinline__ void
i8_results(const uint64_t *list, uint32_t m, uint32_t k, int64_t *ids, float *scores)
{
	for (uint32_t i = threadIdx.x; i < k; i += NT)
	{
		ids[i] = i < m ? (int64_t) (uint32_t) list[i] : -1;
		scores[i] = i < m ? i8_word_score(list[i]) : I8_NINF;
	}
}

/*
 * One block of threads takes a query from its maxima to its results where its candidates fit LDS (k <= 128) and either
 * there are blocks for the whole chip or a query's picked rows are few bytes (50 x 300007 x 1536, k 100: the whole search
 * 149 us in parts, 220 so).  Bound by latency, step after step: one query over 10 k x 128 7 us, 1024 over 1M x 768 63.
 */
#define I8_FUSED_K 128
#define I8_FUSED_BYTES (512u << 10)

template <int NT>
__global__ __launch_bounds__(NT) void
k_i8_finish(const unsigned char *__restrict__ rows, const unsigned char *__restrict__ queries, uint32_t kp, I8Out o, uint32_t k,
			int64_t *__restrict__ ids, float *__restrict__ scores)
{
	__shared__ I8Select<NT, 512> S;
	__shared__ uint32_t picked[512];			/* (quads first) */
	__shared__ int sum[I8_FUSED_K * 32];		/* (a score's bits take the place of its sum) */
	const uint32_t q = blockIdx.x;
	const float qs = o.qscale[q];
	const uint32_t kk = i8_pick(S, picked, o.gmax + (size_t) q * o.ngp, o.qmax + (size_t) q * (o.ngp / 4), (o.n + 31) / 32, k);
	const float floor = kk == k ? i8_word_score(S.list[k - 1]) : I8_NINF;
	const uint32_t parts = (kp + 32 * I8_PART - 1) / (32 * I8_PART);

	for (uint32_t i = threadIdx.x; i < kk; i += NT)
		picked[i] = (uint32_t) S.list[i];
	for (uint32_t i = threadIdx.x; i < kk * 32; i += NT)
		sum[i] = 0;
	__syncthreads();
	I8Row		first = {};

	if (threadIdx.x < kk * 32)
		first = i8_row(o, picked[threadIdx.x / 32], threadIdx.x % 32, q);
	for (uint32_t item = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); item < kk * parts; item += NT / 64)
	{
		const uint32_t slot = item / parts;
		const int	s = i8_part_sum(rows, queries, kp, picked[slot], q, item - slot * parts);

		if ((threadIdx.x & 63) < 32)
			atomicAdd(&sum[slot * 32 + (threadIdx.x & 31)], s);
	}
	__syncthreads();
	for (uint32_t i = threadIdx.x; i < kk * 32; i += NT)
		sum[i] = __float_as_int(i8_row_score(o, i == threadIdx.x ? first : i8_row(o, picked[i / 32], i % 32, q), sum[i], qs));
	__syncthreads();
	const uint32_t m = i8_select(S, [&](uint32_t i, float &v, uint32_t &id) -> bool {
		v = __int_as_float(sum[i]);
		id = picked[i / 32] * 32 + i % 32;
		return v > I8_NINF;
	}, kk * 32, k, floor);

	i8_results<NT>(S.list, m, k, ids + (size_t) q * k, scores + (size_t) q * k);
}

/* otherwise every picked block of rows has a block of threads of its own (50 x 300007 x 1536, k 100: 9 us to pick, 35 to score
 * 246 MB again, 6 for the best) */
#define I8_NT 1024

__global__ __launch_bounds__(I8_NT) void
k_i8_pick(I8Out o, uint32_t k, uint32_t *__restrict__ picked, uint32_t *__restrict__ npicked, float *__restrict__ floors)
{
	__shared__ I8Select<I8_NT, 2048> S;
	__shared__ uint32_t quads[2048];
	const uint32_t q = blockIdx.x;
	const uint32_t kk = i8_pick(S, quads, o.gmax + (size_t) q * o.ngp, o.qmax + (size_t) q * (o.ngp / 4), (o.n + 31) / 32, k);

	for (uint32_t i = threadIdx.x; i < kk; i += I8_NT)
		picked[(size_t) q * k + i] = (uint32_t) S.list[i];
	if (threadIdx.x == 0)
	{
		npicked[q] = kk;
		floors[q] = kk == k ? i8_word_score(S.list[k - 1]) : I8_NINF;
	}
}

__global__ __launch_bounds__(256) void
k_i8_rescore(const unsigned char *__restrict__ rows, const unsigned char *__restrict__ queries, uint32_t kp, I8Out o, uint32_t k,
			 const uint32_t *__restrict__ picked, const uint32_t *__restrict__ npicked, float *__restrict__ cand)
{
	__shared__ int sum[32];
	const uint32_t slot = blockIdx.x, q = blockIdx.y, i = threadIdx.x & 63;

	if (slot >= npicked[q])
		return;
	const uint32_t rb = picked[(size_t) q * k + slot];
	const uint32_t parts = (kp + 32 * I8_PART - 1) / (32 * I8_PART);
	I8Row		w = {};

	if (threadIdx.x < 32)
	{
		sum[i] = 0;
		w = i8_row(o, rb, i, q);
	}
	__syncthreads();
	int			s = 0;

	for (uint32_t part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); part < parts; part += 4)
		s += i8_part_sum(rows, queries, kp, rb, q, part);
	if (i < 32)
		atomicAdd(&sum[i], s);
	__syncthreads();
	if (threadIdx.x < 32)
		cand[((size_t) q * k + slot) * 32 + i] = i8_row_score(o, w, sum[i], o.qscale[q]);
}

__global__ __launch_bounds__(I8_NT) void
k_i8_best(const float *__restrict__ cand, const uint32_t *__restrict__ picked, const uint32_t *__restrict__ npicked,
		  const float *__restrict__ floors, uint32_t k, int64_t *__restrict__ ids, float *__restrict__ scores)
{
	__shared__ I8Select<I8_NT, 2048> S;
	const uint32_t q = blockIdx.x;
	const float *c = cand + (size_t) q * k * 32;
	const uint32_t *p = picked + (size_t) q * k;
	const uint32_t m = i8_select(S, [&](uint32_t i, float &v, uint32_t &id) -> bool {
		v = c[i];
		id = p[i / 32] * 32 + i % 32;
		return v > I8_NINF;
	}, npicked[q] * 32, k, floors[q]);

	i8_results<I8_NT>(S.list, m, k, ids + (size_t) q * k, scores + (size_t) q * k);
}

__global__ __launch_bounds__(256) void
k_i8_none(int64_t *__restrict__ ids, float *__restrict__ scores, uint64_t n)
{
	const uint64_t i = (uint64_t) blockIdx.x * 256 + threadIdx.x;

	if (i < n)
	{
		ids[i] = -1;
		scores[i] = I8_NINF;
	}
}

/* ================================================================== */
/* scores: penalties, biases, masks                                    */
/* ================================================================== */

/* (the runtime copies a launch's arguments one by one, at 70 ns each: fourteen of them 3.5 us, as one 2.6) */
struct I8Adjust
{
	const void *scores;
	int64_t		stride, n;
	const int64_t *seen_off;
	const int32_t *seen_ids;
	int64_t		nseen;
	const float *penalties, *bias;
	int64_t		bias_stride;
	const uint32_t *mask;
	int64_t		mask_stride;
	void	   *out;
	int64_t		ostride;
	int			nq, q0;
};

/*
 * A block of threads takes 256 * VEC * U neighbouring columns of one query and reads their scores at once; meanwhile it counts how
 * often the query's list names each of them (the whole list is read per block: it is short next to the columns, and
 * LDS counters need neither a sort nor a hash nor a bound on its length).  Bound by HBM: a score read and written, a bit
 * of mask (64 x 1M fp32: 122 us, 4.3 TB/s).  Without lists (SEEN false) nothing is shared by a block's columns, and a thread takes
 * one piece: 64 x 333333 and a bias, which the last level cache holds, 38.2 us with four pieces and the counters' LDS, 35.0 with two,
 * 31.6 with one (torch's addition 32.6), 64 x 1M 107.7, 106.9, 105.4, in 16 bits 80, 76, 71; it loses where blocks have little to do
 * (2048 x 3001 and mask and bias: 8.7 -> 9.3).
 */
template <class T, int U, bool SEEN>
__global__ __launch_bounds__(256) void
k_scores_adjust(const I8Adjust a)
{
	constexpr int VEC = 16 / sizeof(T), COLS = 256 * VEC * U;
	__shared__ __attribute__((aligned(16))) uint32_t cnt[SEEN ? COLS : 4];
	const int64_t q = a.q0 + (int64_t) blockIdx.y;
	const int64_t c0 = (int64_t) blockIdx.x * COLS;
	const int	m = (int) min((int64_t) COLS, a.n - c0);
	const T    *src = (const T *) a.scores + q * a.stride + c0;
	T		   *dst = (T *) a.out + q * a.ostride + c0;
	const float *bv = a.bias ? a.bias + q * a.bias_stride + c0 : nullptr;
	const uint32_t *mv = a.mask ? a.mask + q * a.mask_stride + c0 / 32 : nullptr;
	I8Vec<T, VEC> v[U];
	float		add[U][VEC];
	uint32_t	word[U];

#pragma unroll
	for (int u = 0; u < U; u++)
	{
		const int	e = (u * 256 + threadIdx.x) * VEC;

		word[u] = 0xFFFFFFFFu;
		if (e < m)
		{
			if (e + VEC <= m)
				v[u] = i8_get<T, VEC>(src + e);
			else
#pragma unroll
				for (int i = 0; i < VEC; i++)
					if (e + i < m)
						v[u].v[i] = src[e + i];
			if (mv)
				word[u] = mv[e / 32] >> (e % 32);
			if (bv && e + VEC <= m)
#pragma unroll
				for (int i = 0; i < VEC; i += 4)
				{
					const I8Vec<float, 4> b = i8_get<float, 4>(bv + e + i);

#pragma unroll
					for (int j = 0; j < 4; j++)
						add[u][i + j] = b.v[j];
				}
			else if (bv)
#pragma unroll
				for (int i = 0; i < VEC; i++)
					add[u][i] = e + i < m ? bv[e + i] : 0.0f;
		}
	}
	const int64_t lo = SEEN ? max(a.seen_off[q], (int64_t) 0) : 0, hi = SEEN ? min(a.seen_off[q + 1], a.nseen) : 0;
	const bool	seen = hi > lo;
	float		repeat = 1.0f, presence = 0.0f, frequency = 0.0f;

	if (seen)
	{
		repeat = a.penalties[3 * q];
		presence = a.penalties[3 * q + 1];
		frequency = a.penalties[3 * q + 2];
		for (int i = threadIdx.x * 4; i < COLS; i += 1024)
			*(uint4 *) &cnt[i] = make_uint4(0, 0, 0, 0);
		__syncthreads();
		for (int64_t i = lo + threadIdx.x; i < hi; i += 256)
		{
			const int64_t at = (int64_t) a.seen_ids[i] - c0;

			if (at >= 0 && at < m)
				atomicAdd(&cnt[at], 1u);
		}
		__syncthreads();
	}
#pragma unroll
	for (int u = 0; u < U; u++)
	{
		const int	e = (u * 256 + threadIdx.x) * VEC;

		if (e >= m)
			break;
		uint32_t	c[VEC], any = 0;

#pragma unroll
		for (int i = 0; i < VEC; i++)
			c[i] = 0;
		if (seen)
#pragma unroll
			for (int i = 0; i < VEC; i += 4)
			{
				*(uint4 *) &c[i] = *(const uint4 *) &cnt[e + i];
				any |= c[i] | c[i + 1] | c[i + 2] | c[i + 3];
			}
		float		s[VEC];

#pragma unroll
		for (int i = 0; i < VEC; i++)
			s[i] = I8Elem<T>::load(v[u].v[i]);
		if (any)
#pragma unroll
			for (int i = 0; i < VEC; i++)
				if (c[i] > 0)
				{
					s[i] = s[i] > 0.0f ? s[i] / repeat : s[i] * repeat;
					s[i] = s[i] - (presence + (float) c[i] * frequency);
				}
#pragma unroll
		for (int i = 0; i < VEC; i++)
		{
			if (bv)
				s[i] = s[i] + add[u][i];
			if (!(word[u] >> i & 1u))
				s[i] = I8_NINF;
			v[u].v[i] = I8Elem<T>::store(s[i]);
		}
		if (e + VEC <= m)
			i8_put(dst + e, v[u]);
		else
#pragma unroll
			for (int i = 0; i < VEC; i++)
				if (e + i < m)
					dst[e + i] = v[u].v[i];
	}
}

/* ================================================================== */
/* host                                                                */
/* ================================================================== */

/* The library's device for as long as a call runs, and the caller's own again behind it: calls on torch tensors come from
 * programs that keep HIP's current device for themselves. */
struct I8Device
{
	int			callers = -1;
	int enter()
	{
		if (g.inited && hipGetDevice(&callers) != hipSuccess)
			callers = -1;
		return need_init();
	}
	~I8Device()
	{
		if (callers >= 0 && callers != g.device)
			(void) hipSetDevice(callers);
	}
};

/* what a search of host arrays works in on the device */
struct I8Host
{
	char	   *d;
	size_t		bytes;
	bool		busy;
	I8Host	   *next;
};

struct ndbhip_i8
{
	mutable std::mutex host_mtx;
	mutable I8Host *host = nullptr;		/* kept for the next search, one for each that ran at the same time */
	int			dim = 0;
	uint32_t	kp = 0;			/* dimensions, padded */
	int64_t		n = 0;			/* rows */
	int64_t		np = 0;			/* rows laid out */
	unsigned char *d_codes = nullptr;
	float	   *d_scales = nullptr;
};

#define I8_MAX_DIM	32767
#define I8_MAX_ROWS	((int64_t) 0x7FFFFF00)

static int
i8_type_size(int dtype)
{
	return dtype == NDBHIP_F32 ? 4 : dtype == NDBHIP_F16 || dtype == NDBHIP_BF16 ? 2 : dtype == NDBHIP_I8 ? 1 : 0;
}

/* lanes for a row of `units` lane-loads, as a power of two's exponent: the smallest that covers it, at most a wave */
static int
i8_lanes_log2(int64_t units)
{
	int			l = 0;

	while (l < 6 && (1 << l) < units)
		l++;
	return l;
}

/* rows a launch takes: HIP counts a grid's threads in 32 bits, and a thread of these kernels takes at least four bytes of a row */
static int64_t
i8_slab_rows(int dim)
{
	return std::max<int64_t>(I8_ROW_PAD, ((int64_t) 1 << 30) / i8_up((uint32_t) dim, I8_DIM_PAD) / I8_ROW_PAD * I8_ROW_PAD);
}

/* short rows are quantised four (two) a lane at a time where one a lane makes six blocks a compute unit (us: 100000 x 16 fp32, 6.1
 * blocks 4.1 -> 3.8, 1M x 128 177 -> 113; 10000 x 128, 4.9 blocks 3.7 -> 4.2, 1000 x 128 2.8 -> 3.9) */
static bool
i8_many(int64_t nrows, int lanes_log2)
{
	return nrows >> (8 - lanes_log2) >= (int64_t) g.num_cus * 6;
}

template <class T, bool BLOCKED>
static int
i8_quantize_launch(const void *d_x, int64_t nrows, int64_t nrows_out, int dim, int64_t xstride, unsigned char *codes, int64_t cstride,
				   uint32_t kp, float *scales)
{
	constexpr int VEC = 16 / sizeof(T);
	const int	ll = i8_lanes_log2((dim + VEC - 1) / VEC);
	const int64_t slab = i8_slab_rows(dim);

	for (int64_t r0 = 0; r0 < nrows_out; r0 += slab)
	{
		const int64_t m = std::min(slab, nrows_out - r0), real = std::max<int64_t>(0, std::min(m, nrows - r0));

		/* (a launch of padding rows alone reads nothing; its pointer stays at the first row) */
		auto		launch = [&](auto kernel, int rows) {
			const int64_t per = (256 >> ll) * rows;

			hipLaunchKernelGGL(kernel, dim3((unsigned) ((m + per - 1) / per)), dim3(256), 0, g.stream,
							   (const T *) d_x + (real ? r0 * xstride : 0), real, m, dim, xstride, ll,
							   codes + r0 * (BLOCKED ? (int64_t) kp : cstride), cstride, kp, scales + r0);
		};

		if constexpr (!BLOCKED)
			if (i8_many(m, ll) && dim <= 2 * VEC << ll)
			{
				if (dim <= VEC << ll)
					launch(k_i8_quantize<T, false, 1, 4>, 4);
				else
					launch(k_i8_quantize<T, false, 2, 2>, 2);
				continue;
			}
		launch(k_i8_quantize<T, BLOCKED, 4, 1>, 1);
	}
	HIP_TRY(hipGetLastError());
	return NDBHIP_OK;
}

/* rows of any input type -> block layout (or rows of bytes) */
template <bool BLOCKED>
static int
i8_quantize_any(const void *d_x, int dtype, int64_t nrows, int64_t nrows_out, int dim, int64_t xstride, unsigned char *codes, int64_t cstride,
				uint32_t kp, float *scales)
{
	if (dtype == NDBHIP_F32)
		return i8_quantize_launch<float, BLOCKED>(d_x, nrows, nrows_out, dim, xstride, codes, cstride, kp, scales);
	if (dtype == NDBHIP_F16)
		return i8_quantize_launch<__half, BLOCKED>(d_x, nrows, nrows_out, dim, xstride, codes, cstride, kp, scales);
	return i8_quantize_launch<__hip_bfloat16, BLOCKED>(d_x, nrows, nrows_out, dim, xstride, codes, cstride, kp, scales);
}

static int
i8_pack(const void *codes, int64_t stride, const float *scales, int64_t nrows, int64_t nrows_out, int dim, uint32_t kp, unsigned char *dst,
		float *sout)
{
	const int64_t slab = i8_slab_rows(dim);

	for (int64_t r0 = 0; r0 < nrows_out; r0 += slab)
	{
		const int64_t m = std::min(slab, nrows_out - r0), real = std::max<int64_t>(0, std::min(m, nrows - r0));
		const uint64_t units = (uint64_t) m * (kp / 16);

		hipLaunchKernelGGL(k_i8_blocks<true>, dim3((unsigned) ((units + 255) / 256)), dim3(256), 0, g.stream,
						   (const unsigned char *) codes + (real ? r0 * stride : 0), dst + r0 * kp, stride, real, m, dim, kp, scales + (real ? r0 : 0), sout + r0);
	}
	HIP_TRY(hipGetLastError());
	return NDBHIP_OK;
}

extern "C" int
ndbhip_i8_quantize_device(const void *d_x, int dtype, int64_t nrows, int dim, int64_t x_stride, int8_t *d_codes, int64_t codes_stride,
						  float *d_scales)
{
	if (dtype != NDBHIP_F32 && dtype != NDBHIP_F16 && dtype != NDBHIP_BF16)
		return fail(NDBHIP_ERR_INVALID, "rows to quantise must be NDBHIP_F32, _F16 or _BF16");
	if (nrows < 0 || nrows > I8_MAX_ROWS || dim < 1 || dim > I8_MAX_DIM || x_stride < dim || codes_stride < dim)
		return fail(NDBHIP_ERR_INVALID, "bad sizes");
	if (nrows > 0 && (!d_x || !d_codes || !d_scales))
		return fail(NDBHIP_ERR_INVALID, "NULL pointer");
	I8Device	dev;

	if (dev.enter()) return NDBHIP_ERR_NODEVICE;
	if (nrows == 0)
		return NDBHIP_OK;
	return i8_quantize_any<false>(d_x, dtype, nrows, nrows, dim, x_stride, (unsigned char *) d_codes, codes_stride, 0, d_scales);
}

template <class T>
static void
i8_dequantize_launch(const int8_t *codes, int64_t cstride, const float *scales, int64_t nrows, int dim, void *out, int64_t ostride)
{
	constexpr int VEC = 16 / sizeof(T);
	const int	ll = i8_lanes_log2((dim + VEC - 1) / VEC);
	const int64_t slab = i8_slab_rows(dim);

	for (int64_t r0 = 0; r0 < nrows; r0 += slab)
	{
		const int64_t m = std::min(slab, nrows - r0);
		auto		launch = [&](auto kernel, int rows) {
			const int64_t per = (256 >> ll) * rows;

			hipLaunchKernelGGL(kernel, dim3((unsigned) ((m + per - 1) / per)), dim3(256), 0, g.stream, codes + r0 * cstride, cstride,
							   scales + r0, m, dim, ll, (T *) out + r0 * ostride, ostride);
		};

		auto		form = [&](auto tail) {
			constexpr bool TAIL = decltype(tail)::value;

			/* (several short rows a lane pay at any number of them: 1000 x 128 fp32 2.5 -> 2.1 us, 1M x 128 189 -> 114) */
			if (dim <= VEC << ll)
				launch(k_i8_dequantize<T, TAIL, 1, 4>, 4);
			else if (dim <= 2 * VEC << ll)
				launch(k_i8_dequantize<T, TAIL, 2, 2>, 2);
			else
				launch(k_i8_dequantize<T, TAIL, 4, 1>, 1);
		};

		if (dim % VEC)
			form(std::true_type{});
		else
			form(std::false_type{});
	}
}

extern "C" int
ndbhip_i8_dequantize_device(const int8_t *d_codes, int64_t codes_stride, const float *d_scales, int64_t nrows, int dim, void *d_out,
							int dtype, int64_t out_stride)
{
	if (dtype != NDBHIP_F32 && dtype != NDBHIP_F16 && dtype != NDBHIP_BF16)
		return fail(NDBHIP_ERR_INVALID, "values must be NDBHIP_F32, _F16 or _BF16");
	if (nrows < 0 || nrows > I8_MAX_ROWS || dim < 1 || dim > I8_MAX_DIM || codes_stride < dim || out_stride < dim)
		return fail(NDBHIP_ERR_INVALID, "bad sizes");
	if (nrows > 0 && (!d_codes || !d_scales || !d_out))
		return fail(NDBHIP_ERR_INVALID, "NULL pointer");
	I8Device	dev;

	if (dev.enter()) return NDBHIP_ERR_NODEVICE;
	if (nrows == 0)
		return NDBHIP_OK;
	if (dtype == NDBHIP_F32)
		i8_dequantize_launch<float>(d_codes, codes_stride, d_scales, nrows, dim, d_out, out_stride);
	else if (dtype == NDBHIP_F16)
		i8_dequantize_launch<__half>(d_codes, codes_stride, d_scales, nrows, dim, d_out, out_stride);
	else
		i8_dequantize_launch<__hip_bfloat16>(d_codes, codes_stride, d_scales, nrows, dim, d_out, out_stride);
	HIP_TRY(hipGetLastError());
	return NDBHIP_OK;
}

extern "C" int
ndbhip_i8_create(int dim, ndbhip_i8 **out)
{
	if (!out)
		return fail(NDBHIP_ERR_INVALID, "out is NULL");
	if (dim < 1 || dim > I8_MAX_DIM)
		return fail(NDBHIP_ERR_INVALID, "dim must be 1 .. %d", I8_MAX_DIM);
	ndbhip_i8  *t = new (std::nothrow) ndbhip_i8();

	if (!t)
		return fail(NDBHIP_ERR_NOMEM, "out of host memory");
	t->dim = dim;
	t->kp = i8_up((uint32_t) dim, I8_DIM_PAD);
	*out = t;
	return NDBHIP_OK;
}

static int
i8_clear(ndbhip_i8 *t)
{
	unsigned char *c = t->d_codes;
	float	   *s = t->d_scales;

	t->d_codes = nullptr;
	t->d_scales = nullptr;
	t->n = t->np = 0;
	while (I8Host *h = t->host)
	{
		t->host = h->next;
		if (h->d)
			(void) hipFree(h->d);
		delete h;
	}
	if (c)
		HIP_TRY(hipFree(c));
	if (s)
		HIP_TRY(hipFree(s));
	return NDBHIP_OK;
}

extern "C" int
ndbhip_i8_destroy(ndbhip_i8 *t)
{
	if (!t)
		return NDBHIP_OK;
	I8Device	dev;

	if (t->d_codes && dev.enter())
		return NDBHIP_ERR_NODEVICE;
	const int	rc = i8_clear(t);

	delete t;
	return rc;
}

/* room for `nrows` rows in place of what the table holds */
static int
i8_room(ndbhip_i8 *t, int64_t nrows)
{
	if (i8_clear(t))
		return NDBHIP_ERR_HIP;
	if (nrows == 0)
		return NDBHIP_OK;
	const int64_t np = (nrows + I8_ROW_PAD - 1) / I8_ROW_PAD * I8_ROW_PAD;
	hipError_t	e = hipMalloc((void **) &t->d_codes, (size_t) np * t->kp);

	if (e == hipSuccess)
		e = hipMalloc((void **) &t->d_scales, (size_t) np * sizeof(float));
	if (e != hipSuccess)
	{
		(void) hipGetLastError();
		(void) i8_clear(t);
		return fail(e == hipErrorOutOfMemory ? NDBHIP_ERR_NOMEM : NDBHIP_ERR_HIP, "no room for %lld rows: %s", (long long) nrows,
					hipGetErrorString(e));
	}
	t->np = np;
	return NDBHIP_OK;
}

extern "C" int
ndbhip_i8_load_device(ndbhip_i8 *t, const void *d_rows, int dtype, int64_t nrows, int64_t row_stride, const float *d_scales)
{
	if (!t)
		return fail(NDBHIP_ERR_INVALID, "table is NULL");
	if (i8_type_size(dtype) == 0)
		return fail(NDBHIP_ERR_INVALID, "rows must be NDBHIP_F32, _F16, _BF16 or _I8");
	if (nrows < 0 || nrows > I8_MAX_ROWS || row_stride < t->dim)
		return fail(NDBHIP_ERR_INVALID, "bad sizes");
	if (nrows > 0 && (!d_rows || (dtype == NDBHIP_I8) != (d_scales != nullptr)))
		return fail(NDBHIP_ERR_INVALID, "rows are NULL, or scales given for rows that are not NDBHIP_I8 (or none for rows that are)");
	I8Device	dev;

	if (dev.enter()) return NDBHIP_ERR_NODEVICE;
	int			rc = i8_room(t, nrows);

	if (rc || nrows == 0)
		return rc;
	if (dtype == NDBHIP_I8)
		rc = i8_pack(d_rows, row_stride, d_scales, nrows, t->np, t->dim, t->kp, t->d_codes, t->d_scales);
	else
		rc = i8_quantize_any<true>(d_rows, dtype, nrows, t->np, t->dim, row_stride, t->d_codes, 0, t->kp, t->d_scales);
	/* (the rows may go once this returns, and the table may be read on any stream) */
	if (!rc && hipStreamSynchronize(g.stream) != hipSuccess)
		rc = fail(NDBHIP_ERR_HIP, "loading an 8-bit table failed");
	if (rc)
		(void) i8_clear(t);
	else
		t->n = nrows;
	return rc;
}

extern "C" int
ndbhip_i8_load(ndbhip_i8 *t, const float *rows, int64_t nrows)
{
	if (!t)
		return fail(NDBHIP_ERR_INVALID, "table is NULL");
	if (nrows < 0 || nrows > I8_MAX_ROWS || (nrows > 0 && !rows))
		return fail(NDBHIP_ERR_INVALID, "bad arguments");
	I8Device	dev;

	if (dev.enter()) return NDBHIP_ERR_NODEVICE;
	int			rc = i8_room(t, nrows);

	if (rc || nrows == 0)
		return rc;
	/* through a device buffer of whole row blocks, so that a table larger than the free memory's half still loads */
	const int64_t slab = std::min<int64_t>(t->np, std::max<int64_t>(I8_ROW_PAD, ((int64_t) 256 << 20) / (4 * t->dim) / I8_ROW_PAD * I8_ROW_PAD));
	float	   *d = nullptr;

	if (hipMalloc((void **) &d, (size_t) std::min(slab, nrows) * t->dim * sizeof(float)) != hipSuccess)
	{
		(void) hipGetLastError();
		(void) i8_clear(t);
		return fail(NDBHIP_ERR_NOMEM, "no room to load through");
	}
	for (int64_t r0 = 0; r0 < nrows && !rc; r0 += slab)
	{
		const int64_t m = std::min(slab, nrows - r0), mp = std::min(slab, t->np - r0);

		if (hipMemcpyAsync(d, rows + r0 * t->dim, (size_t) m * t->dim * sizeof(float), hipMemcpyHostToDevice, g.stream) != hipSuccess)
			rc = fail(NDBHIP_ERR_HIP, "loading an 8-bit table failed");
		else
			rc = i8_quantize_any<true>(d, NDBHIP_F32, m, mp, t->dim, t->dim, t->d_codes + (size_t) r0 * t->kp, 0, t->kp, t->d_scales + r0);
	}
	if (hipStreamSynchronize(g.stream) != hipSuccess && !rc)
		rc = fail(NDBHIP_ERR_HIP, "loading an 8-bit table failed");
	(void) hipFree(d);
	if (rc)
		(void) i8_clear(t);
	else
		t->n = nrows;
	return rc;
}

extern "C" int
ndbhip_i8_export_device(const ndbhip_i8 *t, int8_t *d_codes, int64_t codes_stride, float *d_scales)
{
	if (!t)
		return fail(NDBHIP_ERR_INVALID, "table is NULL");
	if (t->n > 0 && (!d_codes || !d_scales || codes_stride < t->dim))
		return fail(NDBHIP_ERR_INVALID, "bad arguments");
	I8Device	dev;

	if (dev.enter()) return NDBHIP_ERR_NODEVICE;
	if (t->n == 0)
		return NDBHIP_OK;
	const int64_t slab = i8_slab_rows(t->dim);

	for (int64_t r0 = 0; r0 < t->n; r0 += slab)
	{
		const int64_t m = std::min(slab, t->n - r0);
		const uint64_t units = (uint64_t) m * (t->kp / 16);

		hipLaunchKernelGGL(k_i8_blocks<false>, dim3((unsigned) ((units + 255) / 256)), dim3(256), 0, g.stream,
						   (const unsigned char *) t->d_codes + r0 * t->kp, (unsigned char *) d_codes + r0 * codes_stride, codes_stride, m, m, t->dim, t->kp, t->d_scales + r0, d_scales + r0);
	}
	HIP_TRY(hipGetLastError());
	return NDBHIP_OK;
}

extern "C" int64_t
ndbhip_i8_nrows(const ndbhip_i8 *t)
{
	return t ? t->n : -1;
}

extern "C" int
ndbhip_i8_dim(const ndbhip_i8 *t)
{
	return t ? t->dim : -1;
}

/* ------------------------------------------------------------------ */

static size_t
i8_round(size_t b)
{
	return (b + 255) & ~(size_t) 255;
}

/* workspace of a batch of nq queries: their blocks and scales, then what a search leaves between its kernels */
struct I8Ws
{
	uint32_t	nqp, ng, ngp;
	size_t		q_off, qs_off, gm_off, qm_off, pick_off, npick_off, floor_off, cand_off, total;
};

static bool
i8_fused(const ndbhip_i8 *t, int nq, int k)
{
	return k <= I8_FUSED_K && (nq >= g.num_cus || (uint64_t) k * 32 * t->kp <= I8_FUSED_BYTES);
}

static I8Ws
i8_ws(const ndbhip_i8 *t, int nq, int k)
{
	I8Ws		w;
	size_t		at = 0;
	auto		take = [&](size_t b) { const size_t o = at; at += i8_round(b); return o; };

	w.nqp = i8_up((uint32_t) nq, I8_ROW_PAD);
	w.ng = (uint32_t) ((t->n + 31) / 32);
	w.ngp = i8_up(w.ng, 8);
	w.q_off = take((size_t) w.nqp * t->kp);
	w.qs_off = take((size_t) w.nqp * sizeof(float));
	w.gm_off = take(k ? (size_t) nq * w.ngp * sizeof(float) : 0);
	w.qm_off = take(k ? (size_t) nq * (w.ngp / 4) * sizeof(float) : 0);
	/* (what ndbhip_i8_workspace says grows with nq: room for the largest batch that is not fused) */
	const size_t split = k > I8_FUSED_K ? (size_t) nq : i8_fused(t, 1, k) ? 0 : (size_t) std::min(nq, g.num_cus);

	w.pick_off = take(split * k * sizeof(uint32_t));
	w.npick_off = take(split * sizeof(uint32_t));
	w.floor_off = take(split * sizeof(float));
	w.cand_off = take(split * k * 32 * sizeof(float));
	w.total = at;
	return w;
}

/*
 * Queries a call takes at a time: as many as leave its workspace near a gigabyte, and the wide tile's 256 as long as that is
 * no more than 16, in whole tiles; a search leaves 5 bytes a query for 32 rows, which hold 68 each at the least.  (256 queries of
 * 100M x 64, 3.7 GB: 7.8 ms; in passes of 96, 10.9.)  Not below 32, the queries the stream multiplies with one reading of the table.
 */
static int
i8_chunk(const ndbhip_i8 *t, int nq, int k)
{
	const size_t per = (size_t) t->kp + 12 + (k > 0 ? (size_t) (t->n + 255) / 32 * 5 : 0) + (k > I8_FUSED_K ? (size_t) k * 132 : 0);
	const size_t m = std::max({((size_t) 1 << 30) / per, std::min<size_t>(((size_t) 16 << 30) / per, 256), (size_t) 32});

	return (int) std::min<size_t>((size_t) nq, std::min<size_t>(m >= 256 ? m / 256 * 256 : m / 32 * 32, 4096));
}

extern "C" int
ndbhip_i8_workspace(const ndbhip_i8 *t, int nq, int k, size_t *bytes)
{
	if (!t || !bytes)
		return fail(NDBHIP_ERR_INVALID, "NULL pointer");
	if (nq < 0 || k < 0 || k > NDBHIP_MAX_K)
		return fail(NDBHIP_ERR_INVALID, "bad sizes");
	*bytes = nq == 0 || t->n == 0 ? 0 : i8_ws(t, i8_chunk(t, nq, k), k).total;
	return NDBHIP_OK;
}

static int
i8_check_queries(const ndbhip_i8 *t, const void *d_q, int q_type, const float *d_q_scales, int nq, int64_t q_stride)
{
	if (!t)
		return fail(NDBHIP_ERR_INVALID, "table is NULL");
	if (i8_type_size(q_type) == 0)
		return fail(NDBHIP_ERR_INVALID, "queries must be NDBHIP_F32, _F16, _BF16 or _I8");
	if (nq < 0 || q_stride < t->dim)
		return fail(NDBHIP_ERR_INVALID, "bad sizes");
	if (nq > 0 && (!d_q || (q_type == NDBHIP_I8) != (d_q_scales != nullptr)))
		return fail(NDBHIP_ERR_INVALID, "queries are NULL, or scales given for queries that are not NDBHIP_I8 (or none for queries that are)");
	return NDBHIP_OK;
}

static int
i8_check_ws(const ndbhip_i8 *t, int nq, int k, const void *d_ws, size_t ws_bytes)
{
	const size_t want = i8_ws(t, i8_chunk(t, nq, k), k).total;

	if (!d_ws || ws_bytes < want || ((uintptr_t) d_ws & 255))
		return fail(NDBHIP_ERR_INVALID, "the workspace must be %zu bytes on a 256-byte boundary (ndbhip_i8_workspace)", want);
	return NDBHIP_OK;
}

/* a batch's queries into the workspace, as bytes in the block layout */
static int
i8_take_queries(const ndbhip_i8 *t, const void *d_q, int q_type, const float *d_q_scales, int64_t q0, int m, int64_t q_stride, char *ws,
				const I8Ws &w)
{
	const char *q = (const char *) d_q + q0 * q_stride * i8_type_size(q_type);
	unsigned char *codes = (unsigned char *) ws + w.q_off;
	float	   *scales = (float *) (ws + w.qs_off);

	if (q_type == NDBHIP_I8)
		return i8_pack(q, q_stride, d_q_scales + q0, m, w.nqp, t->dim, t->kp, codes, scales);
	return i8_quantize_any<true>(q, q_type, m, w.nqp, t->dim, q_stride, codes, 0, t->kp, scales);
}

template <int NWQ, class KIND>
static void
i8_tile_launch(const ndbhip_i8 *t, const unsigned char *queries, const I8Out &o)
{
	typedef I8Tile<NWQ> TILE;
	const uint32_t nrt = (o.n + 255) / 256, nqt = (o.nq + 32 * TILE::QB - 1) / (32 * TILE::QB);
	/* as many blocks as the compute units hold, in whole rounds of the XCDs, and no more than have a tile: the narrow tile's LDS fits
	 * twice without biases and masks, and so, at two waves a SIMD, do its registers (with one wave a SIMD asked for, it took 316 of 512
	 * and half of the blocks waited for the others to end: 96 x 1M x 64 76 -> 56 us, 384 x 64000 x 768 36 -> 30) */
	const uint32_t per_cu = NWQ == 2 && !KIND::BIAS && !KIND::MASK ? 2 : 1;
	const uint32_t blocks = std::min(((uint32_t) g.num_cus & ~7u) * per_cu, (nrt + 7) / 8 * 8 * nqt);

	hipLaunchKernelGGL((k_i8_tile<NWQ, KIND>), dim3(blocks), dim3(64 * TILE::NW), 0, g.stream, t->d_codes, queries, t->kp, nrt, nqt, o);
}

template <class KIND>
static void
i8_stream_launch(const ndbhip_i8 *t, const unsigned char *queries, const I8Out &o)
{
	const uint32_t nrb = (o.n + 31) / 32, nqb = (o.nq + 31) / 32;

	/* two query blocks: with two row blocks a wave the queries are read half as often, which pays from 64 k rows on (50 x 300007 x
	 * 1536 108 -> 96 us, 40 x 32000 x 768 9.8 -> 11.1) */
	if (nqb == 1)
		hipLaunchKernelGGL((k_i8_stream<1, 1, KIND>), dim3((nrb + 3) / 4), dim3(256), 0, g.stream, t->d_codes, queries, t->kp, nrb, o);
	else if (nrb >= 2048)
		hipLaunchKernelGGL((k_i8_stream<2, 2, KIND>), dim3((nrb + 7) / 8, (nqb + 1) / 2), dim3(256), 0, g.stream, t->d_codes, queries, t->kp,
						   nrb, o);
	else
		hipLaunchKernelGGL((k_i8_stream<1, 2, KIND>), dim3((nrb + 3) / 4, (nqb + 1) / 2), dim3(256), 0, g.stream, t->d_codes, queries, t->kp,
						   nrb, o);
}

/*
 * Up to 64 queries the table's bytes are what counts, and the stream reads them as fast as memory gives them.  Above, a tile pays
 * where there are enough of them to cover its start (scores of fp16, the queries' way to the block layout with them; stream / 128-query
 * tile / 256-query tile in us): 96 x 16000 x 768 12.9 / 13.3 / 16.5, 256 x 16000 x 768 17.6 / 14.4 / 17.8, 96 x 64000 x 64 9.3 / 10.3 /
 * 11.7, 256 x 64000 x 64 14.3 / 13.6 / 13.4.  The wide tile reads the table half as often (256 x 256000 x 768: 136 / 94 / 82) but wants a
 * tile for every compute unit (512 x 16000 x 768: 23.4 / 16.1 / 18.7) and queries to fill it (384 x 64000 x 768: 57 / 30 / 34).  Over 65 to
 * 512 queries x 4000 to 1M rows x 64 to 1536 dimensions the rule is within 8 % of the best of the three, but for 128 x 1M x 64,
 * whose scores are most of the work (67.6 / 82.7 / 100.8).  What goes past the caches is always many tiles.
 */
template <class KIND>
static int
i8_multiply_kind(const ndbhip_i8 *t, const unsigned char *queries, const I8Out &o)
{
	const uint64_t nrt = (o.n + 255) / 256, w128 = (o.nq + 127) / 128, w256 = (o.nq + 255) / 256;
	bool		few = false;

	if constexpr (KIND::MODE != 2)
		if ((few = o.nq <= 64 || nrt * w128 * (t->kp + 128) <= 80000))
			i8_stream_launch<KIND>(t, queries, o);
	if (!few)
	{
		if (nrt * w256 >= (uint32_t) g.num_cus && 10 * w256 * 2 <= 12 * w128)
			i8_tile_launch<4, KIND>(t, queries, o);
		else
			i8_tile_launch<2, KIND>(t, queries, o);
	}
	HIP_TRY(hipGetLastError());
	return NDBHIP_OK;
}

template <class T>
static int
i8_multiply_scores(const ndbhip_i8 *t, const unsigned char *queries, const I8Out &o)
{
	/*
	 * Scores that fill the last level cache (256 MB) push the table out of it.  Stored past the caches they leave it there for the
	 * next batch: back to back, 1024 x 131072 takes 155 -> 125 us at 512 dimensions, 186 -> 150 at 768 and 267 -> 231 at 1536
	 * (fp32; bf16 258 -> 222).  Where nothing is kept it costs a little (three tables in turn 267 -> 277; a table larger than
	 * the cache, 512 x 400000 x 1536 bf16: 362 -> 385), and smaller matrices or short rows lose by it (256 x 131072 x 768
	 * 42 -> 45, 768 x 131072 x 256 83 -> 90).
	 */
	if ((uint64_t) o.nq * o.n * sizeof(T) > ((uint64_t) 192 << 20) && t->kp >= 512 && (uint64_t) t->np * t->kp <= ((uint64_t) 256 << 20))
		return o.bias ? i8_multiply_kind<I8Kind<2, true, false, T>>(t, queries, o) :
			i8_multiply_kind<I8Kind<2, false, false, T>>(t, queries, o);
	return o.bias ? i8_multiply_kind<I8Kind<0, true, false, T>>(t, queries, o) : i8_multiply_kind<I8Kind<0, false, false, T>>(t, queries, o);
}

static int
i8_multiply_maxima(const ndbhip_i8 *t, const unsigned char *queries, const I8Out &o)
{
	if (o.mask)
		return o.bias ? i8_multiply_kind<I8Kind<1, true, true, float>>(t, queries, o) :
			i8_multiply_kind<I8Kind<1, false, true, float>>(t, queries, o);
	return o.bias ? i8_multiply_kind<I8Kind<1, true, false, float>>(t, queries, o) :
		i8_multiply_kind<I8Kind<1, false, false, float>>(t, queries, o);
}

extern "C" int
ndbhip_i8_product_device(const ndbhip_i8 *t, const void *d_q, int q_type, const float *d_q_scales, int nq, int64_t q_stride,
						 const float *d_bias, void *d_out, int out_type, int64_t out_stride, void *d_ws, size_t ws_bytes)
{
	int			rc = i8_check_queries(t, d_q, q_type, d_q_scales, nq, q_stride);

	if (rc)
		return rc;
	if (out_type != NDBHIP_F32 && out_type != NDBHIP_F16 && out_type != NDBHIP_BF16)
		return fail(NDBHIP_ERR_INVALID, "scores must be NDBHIP_F32, _F16 or _BF16");
	if (out_stride < t->n)
		return fail(NDBHIP_ERR_INVALID, "out_stride is smaller than the table's rows");
	if (nq > 0 && t->n > 0 && !d_out)
		return fail(NDBHIP_ERR_INVALID, "out is NULL");
	if (nq > 0 && t->n > 0 && (rc = i8_check_ws(t, nq, 0, d_ws, ws_bytes)))
		return rc;
	I8Device	dev;

	if (dev.enter()) return NDBHIP_ERR_NODEVICE;
	if (nq == 0 || t->n == 0)
		return NDBHIP_OK;
	const int	chunk = i8_chunk(t, nq, 0);
	const int	osz = i8_type_size(out_type);

	for (int64_t q0 = 0; q0 < nq; q0 += chunk)
	{
		const int	m = (int) std::min<int64_t>(chunk, nq - q0);
		const I8Ws	w = i8_ws(t, m, 0);
		I8Out		o = {};

		if ((rc = i8_take_queries(t, d_q, q_type, d_q_scales, q0, m, q_stride, (char *) d_ws, w)))
			return rc;
		o.rscale = t->d_scales;
		o.qscale = (const float *) ((char *) d_ws + w.qs_off);
		o.bias = d_bias;
		o.out = (char *) d_out + q0 * out_stride * osz;
		o.ostride = out_stride;
		o.n = (uint32_t) t->n;
		o.nq = (uint32_t) m;
		const unsigned char *qc = (const unsigned char *) d_ws + w.q_off;

		rc = out_type == NDBHIP_F32 ? i8_multiply_scores<float>(t, qc, o) : out_type == NDBHIP_F16 ? i8_multiply_scores<__half>(t, qc, o) :
			i8_multiply_scores<__hip_bfloat16>(t, qc, o);
		if (rc)
			return rc;
	}
	NDB_STAT_ADD(queries, nq);
	__atomic_fetch_add(&g.host_rows, (uint64_t) nq * t->n, __ATOMIC_RELAXED);
	__atomic_fetch_add(&g.host_bytes, (uint64_t) nq * t->n * t->dim, __ATOMIC_RELAXED);
	return NDBHIP_OK;
}

extern "C" int
ndbhip_i8_search_device(const ndbhip_i8 *t, const void *d_q, int q_type, const float *d_q_scales, int nq, int64_t q_stride,
						const float *d_bias, const uint32_t *d_mask, int64_t mask_stride, int k, int64_t *d_ids, float *d_scores,
						void *d_ws, size_t ws_bytes)
{
	int			rc = i8_check_queries(t, d_q, q_type, d_q_scales, nq, q_stride);

	if (rc)
		return rc;
	if (k < 1 || k > NDBHIP_MAX_K)
		return fail(NDBHIP_ERR_INVALID, "k must be 1 .. %d", NDBHIP_MAX_K);
	if (d_mask && mask_stride != 0 && mask_stride < (t->n + 31) / 32)
		return fail(NDBHIP_ERR_INVALID, "mask_stride must be 0 (one mask) or at least a word for every 32 rows");
	if (nq > 0 && (!d_ids || !d_scores))
		return fail(NDBHIP_ERR_INVALID, "NULL pointer");
	if (nq > 0 && t->n > 0 && (rc = i8_check_ws(t, nq, k, d_ws, ws_bytes)))
		return rc;
	I8Device	dev;

	if (dev.enter()) return NDBHIP_ERR_NODEVICE;
	if (nq == 0)
		return NDBHIP_OK;
	if (t->n == 0)
	{
		const uint64_t all = (uint64_t) nq * k, slab = (uint64_t) 1 << 31;

		/* (HIP counts a grid's threads in 32 bits) */
		for (uint64_t e = 0; e < all; e += slab)
		{
			const uint64_t m = std::min(slab, all - e);

			hipLaunchKernelGGL(k_i8_none, dim3((unsigned) ((m + 255) / 256)), dim3(256), 0, g.stream, d_ids + e, d_scores + e, m);
		}
		HIP_TRY(hipGetLastError());
		return NDBHIP_OK;
	}
	const int	chunk = i8_chunk(t, nq, k);

	for (int64_t q0 = 0; q0 < nq; q0 += chunk)
	{
		const int	m = (int) std::min<int64_t>(chunk, nq - q0);
		const I8Ws	w = i8_ws(t, m, k);
		char	   *ws = (char *) d_ws;
		const unsigned char *qc = (const unsigned char *) ws + w.q_off;
		uint32_t   *picked = (uint32_t *) (ws + w.pick_off), *npicked = (uint32_t *) (ws + w.npick_off);
		float	   *floors = (float *) (ws + w.floor_off), *cand = (float *) (ws + w.cand_off);
		I8Out		o = {};

		if ((rc = i8_take_queries(t, d_q, q_type, d_q_scales, q0, m, q_stride, ws, w)))
			return rc;
		o.rscale = t->d_scales;
		o.qscale = (const float *) (ws + w.qs_off);
		o.bias = d_bias;
		o.mask = d_mask ? d_mask + q0 * mask_stride : nullptr;
		o.mask_stride = mask_stride;
		o.gmax = (float *) (ws + w.gm_off);
		o.qmax = (float *) (ws + w.qm_off);
		o.ngp = w.ngp;
		o.n = (uint32_t) t->n;
		o.nq = (uint32_t) m;
		if ((rc = i8_multiply_maxima(t, qc, o)))
			return rc;
		if (!i8_fused(t, m, k))
		{
			hipLaunchKernelGGL(k_i8_pick, dim3(m), dim3(I8_NT), 0, g.stream, o, (uint32_t) k, picked, npicked, floors);
			hipLaunchKernelGGL(k_i8_rescore, dim3(k, m), dim3(256), 0, g.stream, t->d_codes, qc, t->kp, o, (uint32_t) k, picked,
							   npicked, cand);
			hipLaunchKernelGGL(k_i8_best, dim3(m), dim3(I8_NT), 0, g.stream, cand, picked, npicked, floors, (uint32_t) k, d_ids + q0 * k,
							   d_scores + q0 * k);
		}
		else if (m < g.num_cus)
			hipLaunchKernelGGL(k_i8_finish<1024>, dim3(m), dim3(1024), 0, g.stream, t->d_codes, qc, t->kp, o, (uint32_t) k, d_ids + q0 * k,
							   d_scores + q0 * k);
		else
			hipLaunchKernelGGL(k_i8_finish<256>, dim3(m), dim3(256), 0, g.stream, t->d_codes, qc, t->kp, o, (uint32_t) k, d_ids + q0 * k,
							   d_scores + q0 * k);
		HIP_TRY(hipGetLastError());
	}
	NDB_STAT_ADD(queries, nq);
	__atomic_fetch_add(&g.host_rows, (uint64_t) nq * t->n, __ATOMIC_RELAXED);
	__atomic_fetch_add(&g.host_bytes, (uint64_t) nq * t->n * t->dim, __ATOMIC_RELAXED);
	return NDBHIP_OK;
}

/*
 * hipMalloc and hipFree take their time, and hipFree waits for all work on the device, other threads' too: a table keeps what its
 * searches of host arrays work in, up to a gigabyte each, until its rows go (64 queries of 1M x 768 255 -> 221 us, 1024 1048 -> 910).
 */
#define I8_HOST_KEPT ((size_t) 1 << 30)

static int
i8_host_take(const ndbhip_i8 *t, size_t bytes, I8Host **out)
{
	I8Host	   *take = nullptr;

	{
		std::lock_guard<std::mutex> lk(t->host_mtx);

		/* the smallest that is large enough, else the largest, to be made larger */
		for (I8Host *h = t->host; h; h = h->next)
			if (!h->busy && (!take || (h->bytes >= bytes ? take->bytes < bytes || h->bytes < take->bytes : h->bytes > take->bytes && take->bytes < bytes)))
				take = h;
		if (!take)
		{
			if (!(take = new (std::nothrow) I8Host{nullptr, 0, false, t->host}))
				return fail(NDBHIP_ERR_NOMEM, "out of host memory");
			t->host = take;
		}
		take->busy = true;
	}
	if (take->bytes < bytes)
	{
		if (take->d)
			(void) hipFree(take->d);
		take->d = nullptr;
		take->bytes = 0;
		if (hipMalloc((void **) &take->d, bytes) != hipSuccess)
		{
			(void) hipGetLastError();
			take->d = nullptr;
			std::lock_guard<std::mutex> lk(t->host_mtx);

			take->busy = false;
			return fail(NDBHIP_ERR_NOMEM, "no room for a search (%zu bytes)", bytes);
		}
		take->bytes = bytes;
	}
	*out = take;
	return NDBHIP_OK;
}

static void
i8_host_give(const ndbhip_i8 *t, I8Host *h)
{
	if (h->bytes > I8_HOST_KEPT)
	{
		(void) hipFree(h->d);
		h->d = nullptr;
		h->bytes = 0;
	}
	std::lock_guard<std::mutex> lk(t->host_mtx);

	h->busy = false;
}

/* host queries in, host results out: the shape of ndbhip_ivf_search */
extern "C" int
ndbhip_i8_search(const ndbhip_i8 *t, const float *queries, int nq, const float *bias, const uint32_t *mask, int64_t mask_stride, int k,
				 int64_t *ids, float *scores)
{
	if (!t)
		return fail(NDBHIP_ERR_INVALID, "table is NULL");
	if (nq < 0 || k < 1 || k > NDBHIP_MAX_K)
		return fail(NDBHIP_ERR_INVALID, "bad sizes");
	if (mask && mask_stride != 0 && mask_stride < (t->n + 31) / 32)
		return fail(NDBHIP_ERR_INVALID, "mask_stride must be 0 (one mask) or at least a word for every 32 rows");
	if (nq > 0 && (!queries || !ids || !scores))
		return fail(NDBHIP_ERR_INVALID, "NULL pointer");
	I8Device	dev;

	if (dev.enter()) return NDBHIP_ERR_NODEVICE;
	if (nq == 0)
		return NDBHIP_OK;
	size_t		wsb = 0;
	const size_t qb = (size_t) nq * t->dim * sizeof(float), bb = bias ? (size_t) t->n * sizeof(float) : 0;
	const size_t words = (size_t) (t->n + 31) / 32;
	const size_t mb = !mask ? 0 : (mask_stride ? (size_t) (nq - 1) * mask_stride + words : words) * sizeof(uint32_t);
	const size_t ib = (size_t) nq * k * sizeof(int64_t), sb = (size_t) nq * k * sizeof(float);
	int			rc = ndbhip_i8_workspace(t, nq, k, &wsb);

	if (rc)
		return rc;
	I8Host	   *host;

	if ((rc = i8_host_take(t, i8_round(wsb) + i8_round(qb) + i8_round(bb) + i8_round(mb) + i8_round(ib) + i8_round(sb), &host)))
		return rc;
	char	   *const d = host->d;
	char	   *d_q = d + i8_round(wsb), *d_b = d_q + i8_round(qb), *d_m = d_b + i8_round(bb), *d_i = d_m + i8_round(mb), *d_s = d_i + i8_round(ib);
	bool		ok = hipMemcpyAsync(d_q, queries, qb, hipMemcpyHostToDevice, g.stream) == hipSuccess;

	if (ok && bb)
		ok = hipMemcpyAsync(d_b, bias, bb, hipMemcpyHostToDevice, g.stream) == hipSuccess;
	if (ok && mb)
		ok = hipMemcpyAsync(d_m, mask, mb, hipMemcpyHostToDevice, g.stream) == hipSuccess;
	if (!ok)
		rc = fail(NDBHIP_ERR_HIP, "copying the queries failed");
	if (!rc)
		rc = ndbhip_i8_search_device(t, d_q, NDBHIP_F32, nullptr, nq, t->dim, bb ? (const float *) d_b : nullptr,
									 mb ? (const uint32_t *) d_m : nullptr, mask_stride, k, (int64_t *) d_i, (float *) d_s, d, wsb);
	if (!rc && (hipMemcpyAsync(ids, d_i, ib, hipMemcpyDeviceToHost, g.stream) != hipSuccess ||
				hipMemcpyAsync(scores, d_s, sb, hipMemcpyDeviceToHost, g.stream) != hipSuccess))
		rc = fail(NDBHIP_ERR_HIP, "copying the results failed");
	if (hipStreamSynchronize(g.stream) != hipSuccess && !rc)
		rc = fail(NDBHIP_ERR_HIP, "the search failed");
	i8_host_give(t, host);
	return rc;
}

/* ------------------------------------------------------------------ */

template <class T>
static void
scores_adjust_launch(I8Adjust a)
{
	/* columns a block takes: many scores 4096 (fp32) or 8192 (16 bits), which halves the list's reads; else half of that; without
	 * lists 1024 (2048) */
	constexpr int VEC = 16 / sizeof(T);
	const int	u = !a.seen_off ? 1 : (int64_t) a.nq * a.n >= ((int64_t) 4 << 20) ? 4 : 2, cols = 256 * VEC * u;

	/* (64 bits: behind 2^31 - 65536 queries the next start is not an int) */
	for (int64_t q0 = 0; q0 < a.nq; q0 += 65535)
	{
		const dim3	grid((unsigned) ((a.n + cols - 1) / cols), (unsigned) std::min<int64_t>(65535, a.nq - q0));

		a.q0 = (int) q0;
		if (u == 4)
			hipLaunchKernelGGL((k_scores_adjust<T, 4, true>), grid, dim3(256), 0, g.stream, a);
		else if (u == 2)
			hipLaunchKernelGGL((k_scores_adjust<T, 2, true>), grid, dim3(256), 0, g.stream, a);
		else
			hipLaunchKernelGGL((k_scores_adjust<T, 1, false>), grid, dim3(256), 0, g.stream, a);
	}
}

/* whether an element of nq rows of `row` bytes, `astride` bytes apart, lies among those at b; astride, bstride >= row > 0 */
static bool
i8_overlap(const void *a, int64_t astride, const void *b, int64_t bstride, int nq, int64_t row)
{
	const int64_t d = (int64_t) ((uintptr_t) b - (uintptr_t) a);

	if (d >= (nq - 1) * astride + row || -d >= (nq - 1) * bstride + row)
		return false;
	/* row i of b against the rows of a that start next before it and behind it; equal strides: one row stands for all */
	for (int64_t i = 0; i < (astride == bstride ? 1 : nq); i++)
	{
		const int64_t at = d + i * bstride, j = at >= 0 ? at / astride : -((-at + astride - 1) / astride);

		for (int64_t r = j; r <= j + 1; r++)
			if ((astride == bstride ? r > -nq && r < nq : r >= 0 && r < nq) && at < r * astride + row && r * astride < at + row)
				return true;
	}
	return false;
}

extern "C" int
ndbhip_scores_adjust_device(const void *d_scores, int dtype, int nq, int64_t n, int64_t stride, const int64_t *d_seen_off,
							const int32_t *d_seen_ids, int64_t n_seen, const float *d_penalties, const float *d_bias, int64_t bias_stride,
							const uint32_t *d_mask, int64_t mask_stride, void *d_out, int64_t out_stride)
{
	if (dtype != NDBHIP_F32 && dtype != NDBHIP_F16 && dtype != NDBHIP_BF16)
		return fail(NDBHIP_ERR_INVALID, "scores must be NDBHIP_F32, _F16 or _BF16");
	if (nq < 0 || n < 0 || n > I8_MAX_ROWS || stride < n || out_stride < n)
		return fail(NDBHIP_ERR_INVALID, "bad sizes");
	if (d_bias && bias_stride != 0 && bias_stride < n)
		return fail(NDBHIP_ERR_INVALID, "bias_stride must be 0 (one bias) or at least n");
	if (d_mask && mask_stride != 0 && mask_stride < (n + 31) / 32)
		return fail(NDBHIP_ERR_INVALID, "mask_stride must be 0 (one mask) or at least a word for every 32 scores");
	if (d_seen_off && (n_seen < 0 || !d_seen_ids || !d_penalties))
		return fail(NDBHIP_ERR_INVALID, "offsets without ids or penalties");
	if (nq > 0 && n > 0 && (!d_scores || !d_out))
		return fail(NDBHIP_ERR_INVALID, "NULL pointer");
	if (nq > 1 && d_scores == d_out && stride != out_stride)
		return fail(NDBHIP_ERR_INVALID, "in place, the two strides must be the same");
	if (nq > 0 && n > 0 && d_scores != d_out &&
		i8_overlap(d_scores, (nq > 1 ? stride : n) * i8_type_size(dtype), d_out, (nq > 1 ? out_stride : n) * i8_type_size(dtype), nq,
				   n * i8_type_size(dtype)))
		return fail(NDBHIP_ERR_INVALID, "out and scores overlap");
	I8Device	dev;

	if (dev.enter()) return NDBHIP_ERR_NODEVICE;
	if (nq == 0 || n == 0)
		return NDBHIP_OK;
	const I8Adjust a = {d_scores, stride, n, d_seen_off, d_seen_ids, n_seen, d_penalties, d_bias, bias_stride, d_mask, mask_stride, d_out,
	out_stride, nq, 0};

	if (dtype == NDBHIP_F32)
		scores_adjust_launch<float>(a);
	else if (dtype == NDBHIP_F16)
		scores_adjust_launch<__half>(a);
	else
		scores_adjust_launch<__hip_bfloat16>(a);
	HIP_TRY(hipGetLastError());
	return NDBHIP_OK;
}
