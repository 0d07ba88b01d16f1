// dms_amd/csrc/linear_attention.inl -- the chunked linear recurrence with a scalar decay for each head.
//
//   S_t = a_t S_{t-1} + y_t^T z_t,   o_t = x_t S_t,   a_t = 2^{g_t}
//
// With G the inclusive sum of g inside a chunk of C tokens and S the state before the chunk,
//   o_i = 2^{G_i} x_i S + sum_{j <= i} 2^{G_i - G_j} (x_i . y_j) z_j
//   S'  = 2^{G_C} S + sum_j 2^{G_C - G_j} y_j^T z_j
// Every exponent is a difference of sums that the decay makes <= 0, so nothing overflows whatever the decays are.  G
// is summed in 64 bits and kept as two floats: the difference of two far sums keeps its low bits.
//
// All four products run on the bf16 matrix instruction (16x16x32).  An operand of t bits is the sum of bf16 planes
// (bf16: 1, fp16: 2, fp32: 3; a number that the kernel itself computed, a score or a state: 3 whatever the call's type), and a
// product of two is the sum of the plane products that matter, smallest first, in fp32: 24 bits everywhere, so that
// freezing the decays leaves the other gradients' bits as they are.  Six bf16 products take 96 cycles where the fp32 instruction
// takes 256 for the same product.
//
// A workgroup takes one (sample, head, segment) and walks its chunks with two kinds of waves.  Owners have 16 columns of z each,
// and with them that part of S, which stays in their accumulators from the first chunk to the last: converted, they are the
// operand of the next chunk's x S without any exchange, because the order of a product's inner index is free.  Feeders fetch
// the rows of the chunks to come, lay them into LDS as planes, form decays and scores, and write whole rows of o; transposed
// fragments come from the transposing LDS read.  bf16 chunks have 64 tokens, the others 32 (the planes' room in LDS).
//
// The gradients are the same kernel in other roles: dq on (dO, v, k) forward, dk on (v, dO, q) and dv on (k, q, dO) backward.
//
// Measured (copies here reach 5.1 TB/s): bf16, 512 heads of 64 x 64, 5120 tokens: 360 us, 1.36 GB of inputs and outputs, 3.8 TB/s
// (566 us with one kind of wave that does all; 314 with scores and states of 16 bits, 339 with 24, the rest for what lasting decays
// and sums in the state keep); bf16, 1024 heads, 2000 tokens, all gradients: 990 us for three roles that together read 2.90 GB
// through the L2 (11 tensors of 262 MB) and write 1.06 (3 tensors, the states that meet), 4.0 TB/s; fp32, 160 heads of 100 x 100,
// ragged, up to 2000 tokens: 246 us, of them 73 for the states between segments.  Neither memory nor the matrix units (26 % of the
// cycles in the first case, 20 in the second) nor LDS (45 and 37 %) are full: waves wait for 57 and 62 % of their cycles, most
// at the two barriers a chunk, where owners and feeders meet.
#pragma once
#include "linear_attention.h"

#include <type_traits>

namespace dmn {
namespace la {

typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Kind;      // planes of an operand of the call's type
template <> struct Kind<float> { static constexpr int NP = 3; };
template <> struct Kind<__bf16> { static constexpr int NP = 1; };
template <> struct Kind<_Float16> { static constexpr int NP = 2; };
constexpr int NC = 3;                   // planes of a computed one: scores, states, 2^{G_C - G_j} z_j

// two numbers as sums of N bf16 pairs, each the rounded rest of the ones before it
template <int N>
__device__ __forceinline__ void split2(float x, float y, unsigned (&p)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        p[i] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){x, y}, b16x2));
        if (i + 1 < N) {
            x -= __builtin_bit_cast(float, p[i] << 16);
            y -= __builtin_bit_cast(float, p[i] & 0xffff0000u);
        }
    }
}

// eight numbers as N planes, the operand of a matrix instruction
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], b16x8 (&p)[N])
{
    u32x4 w[N];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        unsigned q[N];
        split2<N>(x[2 * j], x[2 * j + 1], q);
#pragma unroll
        for (int k = 0; k < N; ++k) w[k][j] = q[k];
    }
#pragma unroll
    for (int k = 0; k < N; ++k) p[k] = __builtin_bit_cast(b16x8, w[k]);
}

// The products of planes a[i] b[j] that reach the precision of the finer operand, or of N planes, smallest first: f(i, j) does one
// of them, for all tiles in turn (a matrix instruction that waits for the one before it costs as much as four that do not).
template <int NA, int NB, int N = 1, typename F>
__device__ __forceinline__ void plane_products(F f)
{
    constexpr int L = NA > NB ? NA : NB, M = L > N ? L : N;
#pragma unroll
    for (int s = M - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB) f(i, s - i);
}

__device__ __forceinline__ f32x4 mfma(const b16x8 &a, const b16x8 &b, const f32x4 &c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// The transposing read: in a group of 16 lanes, lane 4j + c names 4 adjacent elements of row j; lane l receives
// element l%4 of the lanes 4j + l/4, j = 0..3.
__device__ __forceinline__ b16x4 read_tr(const __bf16 *p)
{
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    return __builtin_bit_cast(b16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p)));
}

__device__ __forceinline__ b16x8 join(b16x4 a, b16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// A wave-uniform value, kept in scalar registers from here on (left to itself the compiler loads kernel arguments again for
// every chunk, and waits for them).
__device__ __forceinline__ int held(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float held(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); }
__device__ __forceinline__ long long held(long long v)
{
    const unsigned lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return (long long)((unsigned long long)hi << 32 | lo);
}
template <typename P> __device__ __forceinline__ P *held(P *p) { return reinterpret_cast<P *>(held(reinterpret_cast<long long>(p))); }

// Buffer accesses: an offset of NOWHERE reads zero and writes nothing, so rows and columns that do not exist cost no branch.
constexpr unsigned NOWHERE = 0xffffffffu;
constexpr int STREAM = 2;                // non-temporal: whole lines that nobody here reads again do not sit dirty in the L2 at the kernel's end
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void *p)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, 0xfffffff0u, 0x00027000);
}

// Element (row, col) of an LDS tile D elements wide: rows are not padded, their 16-byte pieces are permuted by the row instead.
// With the 64 banks that a read spans, 16 rows at one column and 4 adjacent rows of 16 columns (the transposing read) both
// meet every bank once; rows padded by 16 bytes cost every one of these reads a second turn.
template <int D>
__device__ __forceinline__ int at(int row, int col)
{
    const int f = D == 32 ? 2 * ((row >> 2) & 1) : (D == 64 ? row & 7 : 2 * (row & 7));
    return row * D + ((((col >> 3) ^ f) << 3) | (col & 7));
}

// A tile of C tokens x D elements of one tensor, on its way from memory to LDS: 16 bytes a thread and unit.
// VEC: the pieces that every row's start and width allow (2: 16 bytes, 1: 8 bytes, 0: single elements).
template <typename T, int D, int C, int NTHR, int VEC>
struct Tile {
    static constexpr int UE = 16 / (int)sizeof(T), PER = D / UE, N = C * PER, U = (N + NTHR - 1) / NTHR;
    static constexpr int NP = Kind<T>::NP;
    struct Flight { u32x4 raw[U]; };
    const char *p;             // token 0 of the sample and head
    long long st;              // bytes from token to token
    unsigned off, step;
    int row, dcol, ocol, lds, lds_step;      // ocol: columns of o from the thread's first to the end (drain); lds: of unit 0; the others lie whole multiples of 8 rows from it, so in the same permutation

    // backwards: token t0 + r goes into row C - 1 - r
    __device__ __forceinline__ void init(const Tensor &x, int b, int h, int tid, int reverse)
    {
        p = held(x.p + ((long long)b * x.sb + (long long)(h / x.group) * x.sh) * (int)sizeof(T));
        st = held(x.st * (long long)sizeof(T));
        const int c = (tid % PER) * UE;
        row = tid / PER;
        off = (unsigned)row * (unsigned)st + (unsigned)(c * (int)sizeof(T));
        step = (unsigned)(NTHR / PER) * (unsigned)st;
        dcol = x.d - c;
        static_assert((NTHR / PER) % 8 == 0, "units have to keep the row's permutation");
        lds = at<D>(reverse ? C - 1 - row : row, c);
        lds_step = (reverse ? -1 : 1) * (NTHR / PER) * D;
        if (dcol <= 0 || row >= C) row = 1 << 30;        // behind every token: T <= 2^29, and the units' rows stay far below 2^31
    }
    // tokens t0 .. t0 + n - 1, zeros behind them
    __device__ __forceinline__ void fetch(Flight &f, long long t0, int n) const
    {
        u32x4 (&raw)[U] = f.raw;
        const __amdgpu_buffer_rsrc_t rs = buffer(p + t0 * st);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool ok = row + u * (NTHR / PER) < n;
            const unsigned o = off + u * step;
            if (VEC == 2) {
                raw[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, ok ? o : NOWHERE, 0, 0);
            } else if (VEC == 1) {
                const u32x2 a = __builtin_amdgcn_raw_buffer_load_b64(rs, ok ? o : NOWHERE, 0, 0);
                const u32x2 b = __builtin_amdgcn_raw_buffer_load_b64(rs, ok && UE / 2 < dcol ? o + 8 : NOWHERE, 0, 0);
                raw[u] = (u32x4){a.x, a.y, b.x, b.y};
            } else if (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[u][i] = __builtin_amdgcn_raw_buffer_load_b32(rs, ok && i < dcol ? o + 4 * i : NOWHERE, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned lo = __builtin_amdgcn_raw_buffer_load_b16(rs, ok && 2 * i < dcol ? o + 4 * i : NOWHERE, 0, 0);
                    const unsigned hi = __builtin_amdgcn_raw_buffer_load_b16(rs, ok && 2 * i + 1 < dcol ? o + 4 * i + 2 : NOWHERE, 0, 0);
                    raw[u][i] = lo | hi << 16;
                }
            }
        }
    }
    // rows of o out of LDS, where they lie as a tile does: the 16 bytes that unit u would be stored from (of fp32: 8 in plane 0, 8 in
    // plane 1).  A thread takes what its own next store() overwrites, so nobody has to wait in between.  `o` is o's row base.
    __device__ __forceinline__ void drain(const __bf16 *tile, int tid, const char *o, long long o_st, int n) const
    {
        const __amdgpu_buffer_rsrc_t rs = buffer(o);
        const int row0 = tid / PER;
        const unsigned first = (unsigned)row0 * (unsigned)o_st + (unsigned)((tid % PER) * 16);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (U * NTHR > N && tid + u * NTHR >= N) break;
            const __bf16 *q = tile + lds + u * lds_step;
            u32x4 w;
            if constexpr (sizeof(T) == 4) {
                const u32x2 a = *reinterpret_cast<const u32x2 *>(q), b = *reinterpret_cast<const u32x2 *>(q + C * D);
                w = (u32x4){a.x, a.y, b.x, b.y};
            } else {
                w = *reinterpret_cast<const u32x4 *>(q);
            }
            const bool ok = row0 + u * (NTHR / PER) < n && 0 < ocol;
            const unsigned at = first + u * (NTHR / PER) * (unsigned)o_st;
            if (VEC == 2) {
                __builtin_amdgcn_raw_buffer_store_b128(w, rs, ok ? at : NOWHERE, 0, STREAM);
            } else if (VEC == 1) {
                __builtin_amdgcn_raw_buffer_store_b64((u32x2){w.x, w.y}, rs, ok ? at : NOWHERE, 0, 0);
                __builtin_amdgcn_raw_buffer_store_b64((u32x2){w.z, w.w}, rs, ok && UE / 2 < ocol ? at + 8 : NOWHERE, 0, 0);
            } else if (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i) __builtin_amdgcn_raw_buffer_store_b32((unsigned)w[i], rs, ok && i < ocol ? at + 4 * i : NOWHERE, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    __builtin_amdgcn_raw_buffer_store_b16((unsigned short)(w[i / 2] >> (16 * (i % 2))), rs, ok && i < ocol ? at + 2 * i : NOWHERE, 0, 0);
            }
        }
    }
    // into LDS planes of C rows of D elements; the last thread's units may lie behind the tile
    __device__ __forceinline__ void store(const Flight &f, __bf16 *tile, int tid) const
    {
        const u32x4 (&raw)[U] = f.raw;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (U * NTHR > N && tid + u * NTHR >= N) break;
            __bf16 *q = tile + lds + u * lds_step;
            if constexpr (sizeof(T) == 4) {
                unsigned a[NP], b[NP];
                const f32x4 x = __builtin_bit_cast(f32x4, raw[u]);
                split2<NP>(x[0], x[1], a);
                split2<NP>(x[2], x[3], b);
#pragma unroll
                for (int k = 0; k < NP; ++k) *reinterpret_cast<u32x2 *>(q + k * C * D) = (u32x2){a[k], b[k]};
            } else if constexpr (NP == 1) {
                *reinterpret_cast<u32x4 *>(q) = raw[u];
            } else {
                typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
                const h16x8 h = __builtin_bit_cast(h16x8, raw[u]);
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
                b16x8 w[NP];
                dmn::la::split8<NP>(x, w);
#pragma unroll
                for (int k = 0; k < NP; ++k) *reinterpret_cast<b16x8 *>(q + k * C * D) = w[k];
            }
        }
    }
};

// The decays of a chunk, in the order in which its rows are walked (row r is token r, or C - 1 - r where time runs backwards)
template <int C>
struct alignas(16) Decays {
    float Gh[C], Gl[C];        // G_i as two floats
    float E[C], R[C];          // 2^{G_i} scale_x, 2^{G_C - G_i} scale_z
    float F[C];                // 2^{G_e - G_i}, e the last row of i's 16
    float tot;                 // 2^{G_C}
};

// the log decay of a lane's step: of its token, or backwards of the token after it
template <int C>
__device__ __forceinline__ float fetch_decay(const float *pg, long long gt, int t0, int len, int reverse, int lane)
{
    const int t = reverse ? t0 + C - lane : t0 + lane;
    return lane < C && t < len ? pg[(long long)t * gt] : 0.0f;
}

// 2^x as a float for the decay of a chunk.  It meets the state at every one, where the rounding of a decay that lasts, |x| < 1/2, would
// add up: there `carry`, what the factors so far have left out, goes into the next, and their product stays right to one step.
// 1 + y + (y^2/2 + y^3/6 + ..), y = x ln 2, in two floats: the first term left out is below 2^-27.
__device__ __forceinline__ float chunk_decay(double x, float &carry)
{
    const double y = x * 0.69314718055994530942;
    const float yh = (float)y, one = 1.0f + yh;
    float p = 1.0f / 5040;
    p = __builtin_fmaf(p, yh, 1.0f / 720);
    p = __builtin_fmaf(p, yh, 1.0f / 120);
    p = __builtin_fmaf(p, yh, 1.0f / 24);
    p = __builtin_fmaf(p, yh, 1.0f / 6);
    p = __builtin_fmaf(p, yh, 0.5f);
    const float more = (yh - (one - 1.0f)) + __builtin_fmaf(one, carry, __builtin_fmaf(p, yh * yh, (float)(y - (double)yh))), a = one + more;
    const bool lasts = fabsf(yh) < 0.34657359f;
    carry = lasts ? (more - (a - one)) * fast_rcp(a) : 0.0f;
    return lasts ? a : fast_exp2((float)x);
}

// one wave; returns G_C
template <int C>
__device__ __forceinline__ double decays(float g, int lane, float scale_x, float scale_z, float &carry, Decays<C> &d)
{
    const double G = lane_sums(log2_decay(g));
    const double tot = lane_value(G, C - 1);
    const double ends[4] = {lane_value(G, 15), lane_value(G, 31), lane_value(G, C > 32 ? 47 : 15), lane_value(G, C > 32 ? 63 : 15)};
    const double end = lane < 16 ? ends[0] : lane < 32 ? ends[1] : lane < 48 ? ends[2] : ends[3];
    if (lane < C) {
        const float hi = (float)G;
        d.Gh[lane] = hi;
        d.Gl[lane] = (float)(G - (double)hi);
        d.E[lane] = fast_exp2(hi) * scale_x;
        d.R[lane] = fast_exp2((float)(tot - G)) * scale_z;
        d.F[lane] = fast_exp2((float)(end - G));
        const float a = chunk_decay(tot, carry);
        if (lane == 0) d.tot = a;
    }
    return tot;
}

// Four adjacent elements of a token's row, in and out: rows lr + 16 I of a chunk, columns c0 + 16 n on.
template <typename T, int C, int VEC>
struct Rows {
    char *p;                   // token 0 of the sample and head, or null
    long long st;              // bytes from token to token
    unsigned off, row_step;
    int row, row16, f32, es, cols;     // cols: columns from c0 to the end

    __device__ __forceinline__ Rows(const Tensor &x, int b, int h, int reverse, int lr, int c0)
    {
        f32 = sizeof(T) == 4 ? 0 : held(x.f32);
        es = sizeof(T) == 4 || f32 ? 4 : 2;
        p = held(x.p ? x.p + ((long long)b * x.sb + (long long)(h / x.group) * x.sh) * es : nullptr);
        st = held(x.st * es);
        row = reverse ? C - 1 - lr : lr;
        row16 = reverse ? -16 : 16;
        off = (unsigned)row * (unsigned)st + (unsigned)(c0 * es);
        row_step = (unsigned)row16 * (unsigned)st;
        cols = x.d - c0;
    }
    // n: tokens of the chunk
    __device__ __forceinline__ void store4(__amdgpu_buffer_rsrc_t rs, int n_rows, int I, int n, const f32x4 &x) const
    {
        const bool ok = row + I * row16 < n_rows;
        const unsigned o = off + I * row_step + 16 * n * es;
        const int left = cols - 16 * n;
        if (sizeof(T) == 4 || f32) {
            if (VEC == 2 || (VEC == 1 && sizeof(T) == 2)) {
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), rs, ok && 0 < left ? o : NOWHERE, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = x[i];                // by value: a bit cast of a vector's element names the vector
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), rs, ok && i < left ? o + 4 * i : NOWHERE, 0, 0);
                }
            }
        } else if constexpr (sizeof(T) == 2) {
            typedef T tx4 __attribute__((ext_vector_type(4)));
            typedef unsigned short hx4 __attribute__((ext_vector_type(4)));
            const tx4 w = __builtin_convertvector(x, tx4);
            if (VEC >= 1) {
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, w), rs, ok && 0 < left ? o : NOWHERE, 0, 0);
            } else {
                const hx4 e = __builtin_bit_cast(hx4, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) __builtin_amdgcn_raw_buffer_store_b16(e[i], rs, ok && i < left ? o + 2 * i : NOWHERE, 0, 0);
            }
        }
    }
    // as it lies in memory; value() makes numbers of it, later
    typedef typename std::conditional<sizeof(T) == 4, u32x4, u32x2>::type Raw;
    __device__ __forceinline__ Raw load4(__amdgpu_buffer_rsrc_t rs, int n_rows, int I, int n) const
    {
        const bool ok = row + I * row16 < n_rows;
        const unsigned o = off + I * row_step + 16 * n * es;
        const int left = cols - 16 * n;
        if constexpr (sizeof(T) == 4) {
            if (VEC == 2) return __builtin_amdgcn_raw_buffer_load_b128(rs, ok && 0 < left ? o : NOWHERE, 0, 0);
            Raw x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_raw_buffer_load_b32(rs, ok && i < left ? o + 4 * i : NOWHERE, 0, 0);
            return x;
        } else {
            if (VEC >= 1) return __builtin_amdgcn_raw_buffer_load_b64(rs, ok && 0 < left ? o : NOWHERE, 0, 0);
            Raw x;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const unsigned lo = __builtin_amdgcn_raw_buffer_load_b16(rs, ok && 2 * i < left ? o + 4 * i : NOWHERE, 0, 0);
                const unsigned hi = __builtin_amdgcn_raw_buffer_load_b16(rs, ok && 2 * i + 1 < left ? o + 4 * i + 2 : NOWHERE, 0, 0);
                x[i] = lo | hi << 16;
            }
            return x;
        }
    }
    static __device__ __forceinline__ f32x4 value(const Raw &x)
    {
        if constexpr (sizeof(T) == 4) {
            return __builtin_bit_cast(f32x4, x);
        } else {
            typedef T tx4 __attribute__((ext_vector_type(4)));
            return __builtin_convertvector(__builtin_bit_cast(tx4, x), f32x4);
        }
    }
};

// A plane of the scores P: 32 tokens see nothing behind themselves, so that the first 32 rows of 64 are half as long (with three
// planes two workgroups of 64 x 64 bf16 still share a compute unit).  Row lr of tile row I.
template <int C> constexpr int scores_plane() { return C == 64 ? 32 * (32 + 64) : 32 * 32; }
template <int C> __device__ __forceinline__ int score(int I, int lr, int col)
{
    return I < 2 ? at<32>(I * 16 + lr, col) : 32 * 32 + at<C>((I - 2) * 16 + lr, col);
}

// The part of a chunk that one pass (one Role) does, by its NW waves; x, y, z are LDS tiles of NP planes.
template <typename T, int DC, int DZ, int C, int NW, bool STATE_ONLY>
struct Pass {
    static constexpr int NP = Kind<T>::NP;
    static constexpr int NT = DZ / 16 / NW, CT = C / 16, KT = DC / 16;     // tiles of 16: a wave's columns, tokens, rows of S
    f32x4 S[KT][NT];
    f32x4 O[STATE_ONLY ? 1 : CT][NT];

    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) S[t][n] = (f32x4){0, 0, 0, 0};
    }
    __device__ __forceinline__ void zero_rows()
    {
#pragma unroll
        for (int I = 0; I < CT; ++I)
#pragma unroll
            for (int n = 0; n < NT; ++n) O[I][n] = (f32x4){0, 0, 0, 0};
    }
    // between kernels: in the order of the registers
    __device__ __forceinline__ void save(f32x4 *p) const
    {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) p[(t * NT + n) * 64] = S[t][n];
    }
    __device__ __forceinline__ void resume(const f32x4 *p)
    {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) S[t][n] = p[(t * NT + n) * 64];
    }
    // tile t, row r of S is row 16 t + r
    __device__ __forceinline__ void load_state(const float *p, int dc, int dz, int in_c, int in_z, int z0, int lr, int lg)
    {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = 16 * t + 4 * lg + i, z = z0 + 16 * n + lr;
                    if (c < dc && z < dz) S[t][n][i] = p[c * in_c + z * in_z];
                }
    }
    __device__ __forceinline__ void store_state(float *p, int dc, int dz, int out_c, int out_z, int z0, int lr, int lg, float more) const
    {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = 16 * t + 4 * lg + i, z = z0 + 16 * n + lr;
                    if (c < dc && z < dz) p[c * out_c + z * out_z] = S[t][n][i] * more;
                }
    }

    // 2^{G_i - G_j} (x_i . y_j) scale_p for j <= i, into P[plane][i][j].  16 x 16 tiles, computed transposed: a lane holds one row
    // i and 4 adjacent j.  A diagonal tile takes the exponential of every difference; below it the decay is
    // 2^{G_i - G_e} 2^{G_e - G_j}, e the last token of j's 16, both factors at most 1: one exponential a lane.  The tiles right of
    // a diagonal one that a product 32 wide reads are zeros.
    // Token 32 s + 16 u + 4 g + r of a row of P lies in column 32 s + 8 g + 4 u + r: in the order of the transposing reads of z.
    static __device__ __forceinline__ void keep(__bf16 *P, int I, int J, const f32x4 &p, int lr, int lg)
    {
        unsigned a[NC], b[NC];
        split2<NC>(p[0], p[1], a);
        split2<NC>(p[2], p[3], b);
#pragma unroll
        for (int k = 0; k < NC; ++k)
            *reinterpret_cast<u32x2 *>(P + k * scores_plane<C>() + score<C>(I, lr, 32 * (J / 2) + 8 * lg + 4 * (J % 2))) = (u32x2){a[k], b[k]};
    }
    // the tiles J0 .. J1 of rows I; J1 > I stands for the zeros
    template <int I, int J0, int J1>
    static __device__ __forceinline__ void row_tiles(const __bf16 *x, const __bf16 *y, __bf16 *P, const Decays<C> &d, float scale_p, int lr, int lg)
    {
        constexpr int JE = J1 < I ? J1 : I, NJ = JE - J0 + 1;
        f32x4 p[NJ];
#pragma unroll
        for (int J = 0; J < NJ; ++J) p[J] = (f32x4){0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < DC / 32; ++s) {
            b16x8 xf[NP], yf[NJ][NP];
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                xf[k] = *reinterpret_cast<const b16x8 *>(x + k * C * DC + at<DC>(I * 16 + lr, 32 * s + 8 * lg));
#pragma unroll
                for (int J = 0; J < NJ; ++J) yf[J][k] = *reinterpret_cast<const b16x8 *>(y + k * C * DC + at<DC>((J0 + J) * 16 + lr, 32 * s + 8 * lg));
            }
            plane_products<NP, NP, NC>([&](int i, int j) __attribute__((always_inline)) {
#pragma unroll
                for (int J = 0; J < NJ; ++J) p[J] = mfma(yf[J][i], xf[j], p[J]);
            });
        }
        const float gh = d.Gh[I * 16 + lr], gl = d.Gl[I * 16 + lr];
#pragma unroll
        for (int J = J0; J <= J1; ++J) {
            f32x4 q = {0, 0, 0, 0};
            if (J == I) {
                const f32x4 jh = *reinterpret_cast<const f32x4 *>(&d.Gh[I * 16 + 4 * lg]), jl = *reinterpret_cast<const f32x4 *>(&d.Gl[I * 16 + 4 * lg]);
#pragma unroll
                for (int r = 0; r < 4; ++r) q[r] = 4 * lg + r > lr ? 0.0f : p[J <= JE ? J - J0 : 0][r] * scale_p * fast_exp2((gh - jh[r]) + (gl - jl[r]));
            } else if (J < I) {
                const f32x4 f = *reinterpret_cast<const f32x4 *>(&d.F[J * 16 + 4 * lg]);
                const float row = fast_exp2((gh - d.Gh[J * 16 + 15]) + (gl - d.Gl[J * 16 + 15])) * scale_p;
#pragma unroll
                for (int r = 0; r < 4; ++r) q[r] = p[J <= JE ? J - J0 : 0][r] * (row * f[r]);
            }
            keep(P, I, J, q, lr, lg);
        }
    }
    // dealt out to W waves
    template <int W>
    static __device__ __forceinline__ void scores(const __bf16 *x, const __bf16 *y, __bf16 *P, const Decays<C> &d, float scale_p, int wave, int lr, int lg)
    {
        if constexpr (CT == 4 && W == 4) {
            if (wave == 0) row_tiles<0, 0, 1>(x, y, P, d, scale_p, lr, lg);
            else if (wave == 1) row_tiles<1, 0, 1>(x, y, P, d, scale_p, lr, lg);
            else if (wave == 2) row_tiles<2, 0, 3>(x, y, P, d, scale_p, lr, lg);
            else row_tiles<3, 0, 3>(x, y, P, d, scale_p, lr, lg);
        } else if constexpr (CT == 4) {
            static_assert(W == 2, "2 or 4 waves");
            if (wave == 0) {
                row_tiles<0, 0, 1>(x, y, P, d, scale_p, lr, lg);
                row_tiles<3, 0, 3>(x, y, P, d, scale_p, lr, lg);
            } else {
                row_tiles<1, 0, 1>(x, y, P, d, scale_p, lr, lg);
                row_tiles<2, 0, 3>(x, y, P, d, scale_p, lr, lg);
            }
        } else {
            static_assert(CT == 2, "chunks of 32 or 64");
            if (wave == 0) row_tiles<0, 0, 1>(x, y, P, d, scale_p, lr, lg);
            else if (wave == 1 && W == 2) row_tiles<1, 0, 1>(x, y, P, d, scale_p, lr, lg);
            else if (wave == 1) row_tiles<1, 0, 0>(x, y, P, d, scale_p, lr, lg);
            else if (wave == 2) row_tiles<1, 1, 1>(x, y, P, d, scale_p, lr, lg);
        }
    }

    // O^T = 2^{G_i} S^T x^T.  The accumulators of S, converted, are the operand: slots 4u + i of lane group g are row
    // 32 s + 16 u + 4 g + i of S, and x is read in that order.
    __device__ __forceinline__ void from_state(const __bf16 *x, const Decays<C> &d, int lr, int lg)
    {
#pragma unroll
        for (int I = 0; I < CT; ++I)
#pragma unroll
            for (int n = 0; n < NT; ++n) O[I][n] = (f32x4){0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < DC / 32; ++s) {
            b16x8 st[NT][NC];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = S[2 * s + j / 4][n][j % 4];
                split8<NC>(w, st[n]);
            }
            b16x8 xf[CT][NP];
#pragma unroll
            for (int I = 0; I < CT; ++I)
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    const __bf16 *q = x + k * C * DC;
                    xf[I][k] = join(*reinterpret_cast<const b16x4 *>(q + at<DC>(I * 16 + lr, 32 * s + 4 * lg)),
                                    *reinterpret_cast<const b16x4 *>(q + at<DC>(I * 16 + lr, 32 * s + 16 + 4 * lg)));
                }
            plane_products<NC, NP>([&](int i, int j) __attribute__((always_inline)) {
#pragma unroll
                for (int I = 0; I < CT; ++I)
#pragma unroll
                    for (int n = 0; n < NT; ++n) O[I][n] = mfma(st[n][i], xf[I][j], O[I][n]);
            });
        }
#pragma unroll
        for (int I = 0; I < CT; ++I) {
            const float e = d.E[I * 16 + lr];
#pragma unroll
            for (int n = 0; n < NT; ++n) O[I][n] *= e;
        }
    }

    // by 32 tokens: O^T += z^T P^T, and where the state is wanted S = 2^{G_C} S + y^T (2^{G_C - G_j} z_j)
    template <bool UPDATE>
    __device__ __forceinline__ void from_chunk(const __bf16 *y, const __bf16 *z, const __bf16 *P, const Decays<C> &d, int z0, int lr, int lg)
    {
        const float tot = d.tot;
#pragma unroll
        for (int s = 0; s < C / 32; ++s) {
            b16x8 zs[NT][NC];
            const int row = 32 * s + 4 * lg;           // slots 4u + i of lane group g are token 32 s + 16 u + 4 g + i
            b16x8 zf[NT][NP];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    const __bf16 *q = z + k * C * DZ + at<DZ>(row + lr / 4, z0 + 16 * n + 4 * (lr % 4));
                    zf[n][k] = join(read_tr(q), read_tr(q + 16 * DZ));
                }
            }
            if (!STATE_ONLY) {
                b16x8 pf[CT][NC];
#pragma unroll
                for (int I = 2 * s; I < CT; ++I)
#pragma unroll
                    for (int k = 0; k < NC; ++k) pf[I][k] = *reinterpret_cast<const b16x8 *>(P + k * scores_plane<C>() + score<C>(I, lr, 32 * s + 8 * lg));
                plane_products<NP, NC>([&](int i, int j) __attribute__((always_inline)) {
#pragma unroll
                    for (int I = 2 * s; I < CT; ++I)
#pragma unroll
                        for (int n = 0; n < NT; ++n) O[I][n] = mfma(zf[n][i], pf[I][j], O[I][n]);
                });
            }
            if (!UPDATE) continue;
            const f32x4 r0 = *reinterpret_cast<const f32x4 *>(&d.R[row]), r1 = *reinterpret_cast<const f32x4 *>(&d.R[row + 16]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = (float)zf[n][NP - 1][j];
#pragma unroll
                    for (int k = NP - 2; k >= 0; --k) w[j] += (float)zf[n][k][j];
                    w[j] *= j < 4 ? r0[j % 4] : r1[j % 4];
                }
                split8<NC>(w, zs[n]);
            }
            constexpr int TG = 2;                        // rows of S at a time: with 4 the registers of 16 waves do not do
#pragma unroll
            for (int t0 = 0; t0 < KT; t0 += TG) {
                b16x8 yf[TG][NP];
                f32x4 add[TG][NT];                       // apart from S: every product would round it
#pragma unroll
                for (int t = 0; t < TG; ++t)
#pragma unroll
                    for (int n = 0; n < NT; ++n) add[t][n] = (f32x4){0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < TG; ++t)
#pragma unroll
                    for (int k = 0; k < NP; ++k) {
                        const __bf16 *q = y + k * C * DC + at<DC>(row + lr / 4, 16 * (t0 + t) + 4 * (lr % 4));
                        yf[t][k] = join(read_tr(q), read_tr(q + 16 * DC));
                    }
                plane_products<NP, NC>([&](int i, int j) __attribute__((always_inline)) {
#pragma unroll
                    for (int t = 0; t < TG; ++t)
#pragma unroll
                        for (int n = 0; n < NT; ++n) add[t][n] = mfma(yf[t][i], zs[n][j], add[t][n]);
                });
#pragma unroll
                for (int t = 0; t < TG; ++t)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = S[t0 + t][n][i];
                            S[t0 + t][n][i] = s == 0 ? __builtin_fmaf(x, tot, add[t][n][i]) : x + add[t][n][i];
                        }
            }
        }
    }

    // rows of o into a tile of x's shape, in the call's type (fp32: 8 bytes of 4 elements in plane 0, 8 in plane 1)
    __device__ __forceinline__ void lay_rows(__bf16 *tile, int z0, int lr, int lg) const
    {
#pragma unroll
        for (int I = 0; I < CT; ++I)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                __bf16 *q = tile + at<DZ>(I * 16 + lr, z0 + 16 * n + 4 * lg);
                if constexpr (sizeof(T) == 4) {
                    const u32x4 w = __builtin_bit_cast(u32x4, O[I][n]);
                    *reinterpret_cast<u32x2 *>(q) = (u32x2){w.x, w.y};
                    *reinterpret_cast<u32x2 *>(q + C * DZ) = (u32x2){w.z, w.w};
                } else {
                    typedef T tx4 __attribute__((ext_vector_type(4)));
                    *reinterpret_cast<u32x2 *>(q) = __builtin_bit_cast(u32x2, __builtin_convertvector(O[I][n], tx4));
                }
            }
    }

    // rows of o to memory from the owners' registers: row r is token t0 + r, or t0 + C - 1 - r where time runs backwards
    template <int VEC>
    __device__ __forceinline__ void store_rows(const Rows<T, C, VEC> &o, int t0, int len) const
    {
        const __amdgpu_buffer_rsrc_t rs = buffer(o.p + (long long)t0 * o.st);
#pragma unroll
        for (int I = 0; I < CT; ++I)
#pragma unroll
            for (int n = 0; n < NT; ++n) o.store4(rs, len - t0, I, n, O[I][n]);
    }

    // a wave's share of sum_c W[t, c] o[t, c]: f(I, n) gives W's four numbers; dots[] goes by the token
    template <typename F>
    __device__ __forceinline__ void dot_rows(float *dots, int reverse, int lr, int lg, F f) const
    {
#pragma unroll
        for (int I = 0; I < CT; ++I) {
            float dot = 0.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const f32x4 x = f(I, n);
#pragma unroll
                for (int i = 0; i < 4; ++i) dot += x[i] * O[I][n][i];
            }
            dot += __shfl_xor(dot, 16);
            dot += __shfl_xor(dot, 32);
            if (lg == 0) dots[reverse ? C - 1 - I * 16 - lr : I * 16 + lr] = dot;
        }
    }
};

template <typename T> constexpr int chunk() { return Kind<T>::NP == 1 ? 64 : 32; }       // chunk_tokens()
// waves that own columns of the state, a 16-column tile each (two of them where 128 columns leave the registers for it)
// waves that feed them: as many as own where splitting fp32 rows into planes is most of their work
template <typename T, int DZ> constexpr int feeders() { return DZ == 32 ? 2 : (DZ == 128 && Kind<T>::NP == 3 ? 8 : 4); }
template <typename T, int DZ> constexpr int owners() { return DZ / 16 < 4 ? DZ / 16 : (DZ == 128 ? 8 : 4); }

// rows first .. behind - 1 of o that lie behind the sample's length: zeros
template <typename T>
__device__ __forceinline__ void zero_rows(const Role &ro, int len, int first, int behind, int b, int h, int tid, int nthr)
{
    if (!ro.O.p) return;
    const int r0 = max(first, len), d = ro.O.d;
    for (long long e = tid; e < (long long)(behind - r0) * d; e += nthr) {
        const long long at = (r0 + e / d) * ro.O.st + b * ro.O.sb + h * ro.O.sh + e % d;
        if (ro.O.f32) reinterpret_cast<float *>(ro.O.p)[at] = 0.0f;
        else reinterpret_cast<T *>(ro.O.p)[at] = (T)0.0f;
    }
}

// What one workgroup of a pass works on.
template <int C>
struct Place {
    int bh, seg, ri, b, h, len, live, c0, c1;

    // The roles of a head sit 8 blocks apart: on the same XCD and started together, where they find a little of what the others have
    // read (1024 heads of 64 x 64, 2000 tokens, bf16: 2.90 GB through the L2 and 1321 us in all, 3.14 and 1355 with role after role;
    // 256 heads of 128 x 128: no difference).
    __device__ __forceinline__ Place(const Args &a)
    {
        const int BH = a.B * a.H, per = BH * a.nroles, in = blockIdx.x % per;
        seg = blockIdx.x / per;
        const int eight = in / (8 * a.nroles), left = in % (8 * a.nroles), wide = min(8, BH - 8 * eight);
        ri = left / wide;
        bh = 8 * eight + left % wide;
        b = bh / a.H;
        h = bh % a.H;
        len = __builtin_amdgcn_readfirstlane(valid_length(a.lengths, a.lengths64, b, a.T));
        live = (len + C - 1) / C;                    // chunks with tokens; backwards the first one walked is the partial one
        c0 = seg * a.seg_chunks;
        c1 = min(live, c0 + a.seg_chunks);
    }
};

// The states after each segment but the last, from s_in for the first and from zero for the others.
template <typename T, int DC, int DZ, int VEC>
__global__ void __launch_bounds__((64 * owners<T, DZ>())) state_kernel(const Args a)
{
    constexpr int C = chunk<T>(), NW = owners<T, DZ>(), NTHR = 64 * NW, NP = Kind<T>::NP;
    typedef Pass<T, DC, DZ, C, NW, true> P;
    struct Shared {
        alignas(16) __bf16 y[NP * C * DC];
        alignas(16) __bf16 z[NP * C * DZ];
        Decays<C> d[2];
    };
    __shared__ Shared sm;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, lr = lane & 15, lg = lane >> 4;
    const Place<C> w(a);
    if (w.seg == a.nseg - 1) return;
    const Role &ro = a.role[w.ri];
    const int dc = ro.Y.d, dz = ro.Z.d, z0 = wave * 16 * P::NT, BH = a.B * a.H;
    const float *pg = a.g + w.b * a.gb + w.h * a.gh;
    const auto token0 = [&](int ci) { return (ro.reverse ? w.live - 1 - ci : ci) * C; };
    P ps;
    ps.zero();
    if (w.seg == 0 && ro.s_in) ps.load_state(ro.s_in + (size_t)w.bh * dc * dz, dc, dz, ro.in_c, ro.in_z, z0, lr, lg);
    Tile<T, DC, C, NTHR, VEC> ty;
    Tile<T, DZ, C, NTHR, VEC> tz;
    ty.init(ro.Y, w.b, w.h, tid, ro.reverse);
    tz.init(ro.Z, w.b, w.h, tid, ro.reverse);
    typename decltype(ty)::Flight fy;
    typename decltype(tz)::Flight fz;
    float g = 0.0f, carry = 0.0f;
    double gsum = 0.0;
    const auto fetch = [&](int ci) {
        const int t0 = token0(ci);
        ty.fetch(fy, t0, w.len - t0);
        tz.fetch(fz, t0, w.len - t0);
        if (wave == NW - 1) g = fetch_decay<C>(pg, a.gt, t0, w.len, ro.reverse, lane);
    };
    if (w.c0 < w.c1) fetch(w.c0);
    for (int ci = w.c0; ci < w.c1; ++ci) {
        if (wave == NW - 1) gsum += decays<C>(g, lane, ro.scale_x, ro.scale_z, carry, sm.d[ci & 1]);
        __syncthreads();                              // nobody reads the last chunk's tiles any more
        ty.store(fy, sm.y, tid);
        tz.store(fz, sm.z, tid);
        __syncthreads();
        if (ci + 1 < w.c1) fetch(ci + 1);
        ps.template from_chunk<true>(sm.y, sm.z, nullptr, sm.d[ci & 1], z0, lr, lg);
    }
    f32x4 *const states = reinterpret_cast<f32x4 *>(a.states + ((size_t)(w.ri * BH + w.bh) * a.nseg + w.seg) * (DC * DZ)) + wave * P::KT * P::NT * 64 + lane;
    ps.save(states);
    if (tid == NTHR - 64) a.decays[(size_t)(w.ri * BH + w.bh) * a.nseg + w.seg] = exp2(gsum);
}

// One pass.  The first waves own the state's columns, the others feed them: they fetch and lay out the tiles, keep the
// decays, compute the scores, a chunk ahead, and write the rows of o.  A chunk has two phases, a barrier behind each:
//   1  feeders: o of the last chunk out; x, y, decays of the next one, z of this one    owners: o from the state
//   2  feeders: scores of the next chunk                                               owners: o and the state from this chunk
// so that z alone needs one tile and the owners never wait for the feeders' loads or exponentials.  In phase 2 the owners leave o in the
// x tile that nobody reads any more, and the feeders write whole rows of it (the owners' own columns are 32-byte pieces,
// and cost the memory twice as much).
// Waves of a SIMD that the LDS leaves room for: two workgroups of 8 where the tiles take less than half of it (rows that are
// fetched element by element need the registers more).
template <typename T, int DC, int DZ, int VEC> constexpr int residents()
{
    const int tiles = Kind<T>::NP * chunk<T>() * (4 * DC + DZ) * 2 + 2 * NC * scores_plane<chunk<T>()>() * 2 + 4 * 1024;
    const int waves = owners<T, DZ>() + feeders<T, DZ>();
    return waves / 4 * (VEC && waves == 8 && tiles <= 80 * 1024 ? 2 : 1);
}

// DOTS: the sums of W o as well.
template <typename T, int DC, int DZ, int VEC, bool DOTS>
__global__ void __launch_bounds__((64 * (owners<T, DZ>() + feeders<T, DZ>())), (residents<T, DC, DZ, VEC>())) chunk_kernel(const Args a)
{
    constexpr int C = chunk<T>(), NO = owners<T, DZ>(), NF = feeders<T, DZ>(), NTHR = 64 * (NO + NF);
    constexpr int NP = Kind<T>::NP;
    constexpr bool WHOLE = DC == DZ;                 // rows of o fit x's tile
    constexpr int AHEAD = DC <= 64 && DZ <= 64 ? 2 : 1;   // chunks of rows in flight: with 128 columns one is as many bytes, and registers are short
    typedef Pass<T, DC, DZ, C, NO, false> P;
    struct Shared {
        alignas(16) __bf16 x[2][NP * C * DC];
        alignas(16) __bf16 y[2][NP * C * DC];
        alignas(16) __bf16 z[NP * C * DZ];
        alignas(16) __bf16 p[2][NC * scores_plane<C>()];
        Decays<C> d[2];
        float dots[NO][C];
    };
    __shared__ Shared sm;

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, lr = lane & 15, lg = lane >> 4;
    const Place<C> w(a);
    const Role &ro = a.role[w.ri];
    const int c0 = held(w.c0), c1 = held(w.c1), len = w.len, live = held(w.live), reverse = held(ro.reverse);
    const float *pg = held(a.g + w.b * a.gb + w.h * a.gh);
    float *const dots = held(ro.dots ? ro.dots + (size_t)w.bh * a.T : nullptr);
    const auto token0 = [&](int ci) { return (reverse ? live - 1 - ci : ci) * C; };

    if (wave >= NO) {
        const int fw = wave - NO, ft = tid - 64 * NO;
        Tile<T, DC, C, 64 * NF, VEC> tx, ty;
        Tile<T, DZ, C, 64 * NF, VEC> tz;
        tx.init(ro.X, w.b, w.h, ft, reverse);
        ty.init(ro.Y, w.b, w.h, ft, reverse);
        tz.init(ro.Z, w.b, w.h, ft, reverse);
        struct Chunk {
            typename decltype(tx)::Flight x, y;
            typename decltype(tz)::Flight z;
            float g;
        } even, odd;                                     // the chunks of either parity from c0 on
        const long long gt = held(a.gt), o_st = held(ro.O.st * (long long)sizeof(T));
        const char *const o = held(WHOLE && ro.O.p && (sizeof(T) == 4 || !ro.O.f32) ? ro.O.p + ((long long)w.b * ro.O.sb + (long long)w.h * ro.O.sh) * (long long)sizeof(T) : nullptr);
        tx.ocol = ro.O.d - (ft % tx.PER) * tx.UE;
        const float scale_p = held(ro.scale_p), scale_x = held(ro.scale_x), scale_z = held(ro.scale_z);
        const auto fetch_xy = [&](int ci, Chunk &f) __attribute__((always_inline)) {
            if (ci >= c1) return;
            const int t0 = token0(ci);
            tx.fetch(f.x, t0, len - t0);
            ty.fetch(f.y, t0, len - t0);
            if (fw == 0) f.g = fetch_decay<C>(pg, gt, t0, len, reverse, lane);
        };
        const auto fetch_z = [&](int ci, Chunk &f) __attribute__((always_inline)) {
            if (ci < c1) tz.fetch(f.z, token0(ci), len - token0(ci));
        };
        float carry = 0.0f;
        const auto store_xy = [&](int ci, const Chunk &f) __attribute__((always_inline)) {
            tx.store(f.x, sm.x[ci & 1], ft);
            ty.store(f.y, sm.y[ci & 1], ft);
            if (fw == 0) decays<C>(f.g, lane, scale_x, scale_z, carry, sm.d[ci & 1]);
        };
        const auto flush = [&](int ci) __attribute__((always_inline)) {
            if (o) tx.drain(sm.x[ci & 1], ft, o + token0(ci) * o_st, o_st, len - token0(ci));
            const int t = token0(ci) + ft;
            if (DOTS && dots && ft < C && t < len) {
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < NO; ++i) s += sm.dots[i][ft];
                dots[t] = s;
            }
        };
        const auto lay = [&](int ci, Chunk &mine, Chunk &other) __attribute__((always_inline)) {
            if (ci >= c0) {
                tz.store(mine.z, sm.z, ft);
                fetch_z(ci + AHEAD, mine);
            }
            if (ci + 1 < c1) {
                store_xy(ci + 1, other);
                fetch_xy(ci + 1 + AHEAD, other);
            }
        };
        fetch_xy(c0, even);
        fetch_z(c0, even);
        if (AHEAD == 2) {
            fetch_xy(c0 + 1, odd);
            fetch_z(c0 + 1, odd);
        }
        for (int ci = c0 - 1; ci < c1; ++ci) {           // the first turn lays out chunk c0 only
            if (ci > c0) flush(ci - 1);
            if (AHEAD == 1) lay(ci, even, even);
            else if ((ci - c0) & 1) lay(ci, odd, even);
            else lay(ci, even, odd);
            __syncthreads();
            if (ci + 1 < c1) P::template scores<NF>(sm.x[(ci + 1) & 1], sm.y[(ci + 1) & 1], sm.p[(ci + 1) & 1], sm.d[(ci + 1) & 1], scale_p, fw, lr, lg);
            __syncthreads();
        }
        if (c0 < c1) flush(c1 - 1);
    } else {
        const int dc = ro.Y.d, dz = ro.Z.d, z0 = wave * 16 * P::NT;
        const Rows<T, C, VEC> out(ro.O, w.b, w.h, reverse, lr, z0 + 4 * lg), wrows(DOTS && dots ? ro.W : ro.O, w.b, w.h, reverse, lr, z0 + 4 * lg);
        const bool fresh = w.seg == 0 && !ro.s_in, leaves = ro.s_out && w.seg == a.nseg - 1;
        P ps;
        f32x4 *const keep = reinterpret_cast<f32x4 *>(held(DOTS && ro.keep ? ro.keep + (size_t)w.bh * anchors(a.T) * (DC * DZ) : nullptr));
        ps.zero();
        ps.zero_rows();                                  // for good where the owner has no columns: its dots are 0
        if (w.seg == 0) {
            if (ro.s_in) ps.load_state(ro.s_in + (size_t)w.bh * dc * dz, dc, dz, ro.in_c, ro.in_z, z0, lr, lg);
        } else {
            ps.resume(reinterpret_cast<const f32x4 *>(a.states + ((size_t)(w.ri * a.B * a.H + w.bh) * a.nseg + w.seg - 1) * (DC * DZ)) +
                      wave * P::KT * P::NT * 64 + lane);
        }
        if (c0 <= c1) {                                  // the feeders' first turn
            __syncthreads();
            __syncthreads();
        }
        for (int ci = c0; ci < c1; ++ci) {
            const Decays<C> &d = sm.d[ci & 1];
            const int t0 = token0(ci);
            const int edge = reverse ? t0 : t0 + C;          // the state after this chunk is the one between the tokens edge - 1 and edge
            const bool anchor = DOTS && keep && edge % ANCHOR == 0 && edge > 0 && edge < len;
            typename Rows<T, C, VEC>::Raw wf[DOTS ? P::CT : 1][P::NT];
            if (DOTS && dots) {                              // on their way while o is computed
                const __amdgpu_buffer_rsrc_t rs = buffer(wrows.p + (long long)t0 * wrows.st);
#pragma unroll
                for (int I = 0; I < P::CT; ++I)
#pragma unroll
                    for (int n = 0; n < P::NT; ++n) wf[I][n] = wrows.load4(rs, len - t0, I, n);
            }
            // an owner without columns has nothing to do, the first chunk of a sequence no state to read, the last none to leave
            if (z0 < dz && ci == c0 && fresh) ps.zero_rows();
            else if (z0 < dz) ps.from_state(sm.x[ci & 1], d, lr, lg);
            __syncthreads();
            if (z0 < dz && (ci + 1 < c1 || leaves || anchor)) ps.template from_chunk<true>(sm.y[ci & 1], sm.z, sm.p[ci & 1], d, z0, lr, lg);
            else if (z0 < dz) ps.template from_chunk<false>(sm.y[ci & 1], sm.z, sm.p[ci & 1], d, z0, lr, lg);
            if (WHOLE && !out.f32) ps.lay_rows(sm.x[ci & 1], z0, lr, lg);
            else if (out.p) ps.store_rows(out, t0, len);
            if (__builtin_expect(anchor, 0)) ps.save(keep + (size_t)(edge / ANCHOR - 1) * (DC * DZ / 4) + wave * P::KT * P::NT * 64 + lane);
            if (DOTS && dots)
                ps.dot_rows(sm.dots[wave], reverse, lr, lg, [&](int I, int n) __attribute__((always_inline)) { return Rows<T, C, VEC>::value(wf[I][n]); });
            __syncthreads();
        }
        if (leaves)
            ps.store_state(ro.s_out + (size_t)w.bh * dc * dz, dc, dz, ro.out_c, ro.out_z, z0, lr, lg,
                           ro.last_decay && len > 0 ? fast_exp2((float)log2_decay(pg[0])) : 1.0f);
    }
    zero_rows<T>(ro, len, c0 * C, min(a.T, (c0 + a.seg_chunks) * C), w.b, w.h, tid, NTHR);
}

template <typename T, int DC, int DZ, int VEC>
static int launch_one(const Args &a, int kind, hipStream_t stream)
{
    const unsigned grid = (unsigned)((size_t)a.B * a.H * a.nseg * a.nroles);
    constexpr int n = 64 * (owners<T, DZ>() + feeders<T, DZ>());
    if (kind & STATES) state_kernel<T, DC, DZ, VEC><<<grid, 64 * owners<T, DZ>(), 0, stream>>>(a);
    else if (kind & DOTS_PASS) chunk_kernel<T, DC, DZ, VEC, true><<<grid, n, 0, stream>>>(a);
    else chunk_kernel<T, DC, DZ, VEC, false><<<grid, n, 0, stream>>>(a);
    return launch_status("linear_attention");
}

template <typename T, int VEC>
static int launch_width(const Args &a, int DC, int DZ, int kind, hipStream_t stream)
{
    if (DC == 32) return launch_one<T, 32, 32, VEC>(a, kind, stream);
    if (DC == 64 && DZ == 64) return launch_one<T, 64, 64, VEC>(a, kind, stream);
    if (DC == 64) return launch_one<T, 64, 128, VEC>(a, kind, stream);
    if (DZ == 64) return launch_one<T, 128, 64, VEC>(a, kind, stream);
    return launch_one<T, 128, 128, VEC>(a, kind, stream);
}

template <typename T>
int launch_chunks(const Args &a, int DC, int DZ, int kind, hipStream_t stream)
{
    int vec = 2;                                     // of all rows that the kernel touches
    const auto touch = [&vec](const Tensor &t) { vec = t.p && t.vec < vec ? t.vec : vec; };
    for (int r = 0; r < a.nroles; ++r) {
        touch(a.role[r].Y);
        touch(a.role[r].Z);
        if (kind & STATES) continue;
        touch(a.role[r].X);
        if (a.role[r].dots) touch(a.role[r].W);
        touch(a.role[r].O);
    }
    if (vec == 2) return launch_width<T, 2>(a, DC, DZ, kind, stream);
    if (vec == 1) return launch_width<T, 1>(a, DC, DZ, kind, stream);
    return launch_width<T, 0>(a, DC, DZ, kind, stream);
}

}  // namespace la
}  // namespace dmn
