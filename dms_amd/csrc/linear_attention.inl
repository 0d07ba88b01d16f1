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
// (bf16: 1, fp16: 2, fp32: 3; a number that the kernel itself computed: 2, and 3 beside fp32), and a product of two is
// the sum of the plane products that matter, smallest first, in fp32: 16 bits and more in bf16 and fp16 calls, 24 in
// fp32 ones.  Six bf16 products take 96 cycles where the fp32 instruction takes 256 for the same product.
//
// A workgroup takes one (sample, head, segment) and walks its chunks; a wave owns 16 * NT columns of z, and with them
// that part of S, which stays in its accumulators from the first chunk to the last.  Each accumulator tile holds the
// rows of S in an order that makes it, converted, the operand of the next chunk's x S without any exchange:
// row r of tile t is row 32 (t/2) + 8 (r/4) + 4 (t%2) + r%4 of S.
// x, y, z planes are staged in LDS (rows padded by 16 bytes: 16 rows at one column fall into 64 different banks),
// the next chunk's rows are in flight meanwhile.  Transposed fragments come from the transposing LDS read.
#pragma once
#include "linear_attention.h"

namespace dmn {
namespace la {

typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Kind;      // planes of an operand of the call's type, and of a computed one
template <> struct Kind<float> { static constexpr int NP = 3, NC = 3; };
template <> struct Kind<__bf16> { static constexpr int NP = 1, NC = 2; };
template <> struct Kind<_Float16> { static constexpr int NP = 2, NC = 2; };

template <typename T> struct alignas(16) Row8 { T v[8]; };

// eight elements of a row from column c on, zero behind column d
template <typename T>
__device__ __forceinline__ Row8<T> fetch8(const T *row, int c, int d, int vec)
{
    Row8<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = (T)0.0f;
    if (vec == 2) {
        constexpr int W = 16 / (int)sizeof(T);
        struct alignas(16) V { T v[W]; };
#pragma unroll
        for (int i = 0; i < 8; i += W)
            if (c + i < d) {
                const V t = *reinterpret_cast<const V *>(row + c + i);
#pragma unroll
                for (int j = 0; j < W; ++j) r.v[i + j] = t.v[j];
            }
    } else if (vec == 1) {
        constexpr int W = 8 / (int)sizeof(T);
        struct alignas(8) V { T v[W]; };
#pragma unroll
        for (int i = 0; i < 8; i += W)
            if (c + i < d) {
                const V t = *reinterpret_cast<const V *>(row + c + i);
#pragma unroll
                for (int j = 0; j < W; ++j) r.v[i + j] = t.v[j];
            }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < d) r.v[i] = row[c + i];
    }
    return r;
}

// x as a sum of N bf16 numbers, each the rounded rest of the ones before it
template <int N>
__device__ __forceinline__ void split(float x, __bf16 (&p)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        p[i] = (__bf16)x;
        x -= (float)p[i];
    }
}

template <typename T>
__device__ __forceinline__ void split8(const Row8<T> &r, b16x8 (&p)[Kind<T>::NP])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        __bf16 q[Kind<T>::NP];
        split<Kind<T>::NP>((float)r.v[i], q);
#pragma unroll
        for (int k = 0; k < Kind<T>::NP; ++k) p[k][i] = q[k];
    }
}

// acc += sum of a[i] b[j] over the pairs that reach the precision of the finer operand
template <int NA, int NB>
__device__ __forceinline__ f32x4 mma(const b16x8 (&a)[NA], const b16x8 (&b)[NB], f32x4 acc)
{
    constexpr int M = NA > NB ? NA : NB;
#pragma unroll
    for (int s = M - 1; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], acc, 0, 0, 0);
    return acc;
}

// The transposing read: in a group of 16 lanes, lane 4j + c names 4 adjacent elements of row j; lane l receives
// element l%4 of the lanes 4j + l/4, j = 0..3.
__device__ __forceinline__ b16x4 read_tr(const __bf16 *p)
{
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    return __builtin_bit_cast(b16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p)));
}

template <typename T, int DC, int DZ, int C, bool STATE_ONLY>
struct Shared {
    static constexpr int NP = Kind<T>::NP, NC = Kind<T>::NC;
    static constexpr int LC = DC + 8, LZ = DZ + 8, LP = C + 8;
    alignas(16) __bf16 X[STATE_ONLY ? 1 : NP][STATE_ONLY ? 1 : C][LC];
    alignas(16) __bf16 Y[NP][C][LC];
    alignas(16) __bf16 Z[NP][C][LZ];
    alignas(16) __bf16 P[STATE_ONLY ? 1 : NC][STATE_ONLY ? 1 : C][LP];
    float Gh[C], Gl[C], E[C], R[C];     // G_i as two floats, 2^{G_i}, 2^{G_C - G_i}
    float tot;                          // 2^{G_C}
    float dot[8][C];
};

template <typename T, int DC, int DZ, int C, int NW, bool STATE_ONLY>
__global__ void __launch_bounds__(64 * NW) chunk_kernel(const Args a)
{
    constexpr int NP = Kind<T>::NP, NC = Kind<T>::NC;
    constexpr int NT = DZ / 16 / NW;                 // 16-column tiles of a wave
    constexpr int NTHR = 64 * NW;
    constexpr int UC = (C * DC / 8 + NTHR - 1) / NTHR, UZ = (C * DZ / 8 + NTHR - 1) / NTHR;
    constexpr int CT = C / 16;
    __shared__ Shared<T, DC, DZ, C, STATE_ONLY> sm;

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, lr = lane & 15, lg = lane >> 4;
    const int BH = a.B * a.H;
    const int bh = blockIdx.x % BH, rest = blockIdx.x / BH;
    const int seg = rest % a.nseg, ri = rest / a.nseg;
    if (STATE_ONLY && seg == a.nseg - 1) return;     // the last segment's state is nobody's first
    const Role &ro = a.role[ri];
    const int b = bh / a.H, h = bh % a.H;
    const int len = valid_length(a.lengths, a.lengths64, b, a.T);
    const int dc = ro.Y.d, dz = ro.Z.d;
    const int first = seg * a.seg_chunks * C, behind = min(a.T, first + a.seg_chunks * C);   // steps of this segment
    const int n_live = len > first ? (min(len, behind) - first + C - 1) / C : 0;
    const int zcol0 = wave * 16 * NT;

    const T *px = STATE_ONLY ? nullptr : reinterpret_cast<const T *>(ro.X.p) + b * ro.X.sb + (h / ro.X.group) * ro.X.sh;
    const T *py = reinterpret_cast<const T *>(ro.Y.p) + b * ro.Y.sb + (h / ro.Y.group) * ro.Y.sh;
    const T *pz = reinterpret_cast<const T *>(ro.Z.p) + b * ro.Z.sb + (h / ro.Z.group) * ro.Z.sh;
    const float *pg = a.g + b * a.gb + h * a.gh;

    // ---- the state before the segment
    f32x4 S[DC / 16][NT];
#pragma unroll
    for (int t = 0; t < DC / 16; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) S[t][n] = (f32x4){0, 0, 0, 0};
    const size_t slot = ((size_t)(ri * BH + bh) * a.nseg + seg) * (DC * DZ);
    if (seg == 0) {
        if (ro.s_in) {
            const float *si = ro.s_in + (size_t)bh * dc * dz;
#pragma unroll
            for (int t = 0; t < DC / 16; ++t)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c = 32 * (t / 2) + 8 * lg + 4 * (t % 2) + i, z = zcol0 + 16 * n + lr;
                        if (c < dc && z < dz) S[t][n][i] = si[c * ro.in_c + z * ro.in_z];
                    }
        }
    } else if (!STATE_ONLY) {
        const f32x4 *si = reinterpret_cast<const f32x4 *>(a.states + slot - DC * DZ) + (wave * (DC / 16) * NT) * 64 + lane;
#pragma unroll
        for (int t = 0; t < DC / 16; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) S[t][n] = si[(t * NT + n) * 64];
    }

    // ---- rows in flight
    Row8<T> rx[STATE_ONLY ? 1 : UC], ry[UC], rz[UZ];
    float gnext = 0.0f;
    auto fetch = [&](int s0) {
#pragma unroll
        for (int u = 0; u < UC; ++u) {
            const int e = tid + u * NTHR, r = e / (DC / 8), c = (e % (DC / 8)) * 8, s = s0 + r;
            const bool ok = e < C * DC / 8 && s < len;
            const long long t = ro.reverse ? len - 1 - s : s;
            if (!STATE_ONLY) rx[u] = fetch8<T>(px + t * ro.X.st, ok ? c : 1 << 20, ro.X.d, ro.X.vec);
            ry[u] = fetch8<T>(py + t * ro.Y.st, ok ? c : 1 << 20, ro.Y.d, ro.Y.vec);
        }
#pragma unroll
        for (int u = 0; u < UZ; ++u) {
            const int e = tid + u * NTHR, r = e / (DZ / 8), c = (e % (DZ / 8)) * 8, s = s0 + r;
            const bool ok = e < C * DZ / 8 && s < len;
            const long long t = ro.reverse ? len - 1 - s : s;
            rz[u] = fetch8<T>(pz + t * ro.Z.st, ok ? c : 1 << 20, ro.Z.d, ro.Z.vec);
        }
        if (wave == 0) {
            const int s = s0 + lane;
            gnext = 0.0f;
            if (lane < C && s < len) {
                if (!ro.reverse) gnext = pg[(long long)s * a.gt];
                else if (s > 0) gnext = pg[(long long)(len - s) * a.gt];
            }
        }
    };
    auto flush_dots = [&](int s0) {
        if (tid < C && s0 + tid < len) {
            float d = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) d += sm.dot[w][tid];
            const int s = s0 + tid;
            ro.dots[(size_t)bh * a.T + (ro.reverse ? len - 1 - s : s)] = d;
        }
    };
    double gsum = 0.0;
    if (n_live > 0) fetch(first);

    for (int ci = 0; ci < n_live; ++ci) {
        const int s0 = first + ci * C;
        __syncthreads();                              // nobody reads the last chunk's tiles any more
        if (!STATE_ONLY && ro.dots && ci > 0) flush_dots(s0 - C);
#pragma unroll
        for (int u = 0; u < UC; ++u) {
            const int e = tid + u * NTHR, r = e / (DC / 8), c = (e % (DC / 8)) * 8;
            if (e < C * DC / 8) {
                b16x8 p[NP];
                if (!STATE_ONLY) {
                    split8<T>(rx[u], p);
#pragma unroll
                    for (int k = 0; k < NP; ++k) *reinterpret_cast<b16x8 *>(&sm.X[k][r][c]) = p[k];
                }
                split8<T>(ry[u], p);
#pragma unroll
                for (int k = 0; k < NP; ++k) *reinterpret_cast<b16x8 *>(&sm.Y[k][r][c]) = p[k];
            }
        }
#pragma unroll
        for (int u = 0; u < UZ; ++u) {
            const int e = tid + u * NTHR, r = e / (DZ / 8), c = (e % (DZ / 8)) * 8;
            if (e < C * DZ / 8) {
                b16x8 p[NP];
                split8<T>(rz[u], p);
#pragma unroll
                for (int k = 0; k < NP; ++k) *reinterpret_cast<b16x8 *>(&sm.Z[k][r][c]) = p[k];
            }
        }
        if (wave == 0) {
            double G = log2_decay(gnext);
#pragma unroll
            for (int o = 1; o < C; o <<= 1) {
                const double up = __shfl_up(G, o);
                if (lane >= o) G += up;
            }
            const double tot = __shfl(G, C - 1);
            if (lane < C) {
                const float hi = (float)G;
                sm.Gh[lane] = hi;
                sm.Gl[lane] = (float)(G - (double)hi);
                sm.E[lane] = fast_exp2(hi);
                sm.R[lane] = fast_exp2((float)(tot - G));
                if (lane == 0) sm.tot = fast_exp2((float)tot);
            }
            gsum += tot;
        }
        __syncthreads();
        if (ci + 1 < n_live) fetch(s0 + C);
        const float tot = sm.tot;

        f32x4 O[STATE_ONLY ? 1 : CT][NT];
        if (!STATE_ONLY) {
            // ---- P^T tiles: rows j = the lane's 4 registers, column i = the lane; the 16 x 16 tiles on and below the diagonal
            // go round the waves, and so do the tiles right of a diagonal one that a 32-wide product reads: zeros
            constexpr int NTILE = CT * (CT + 1) / 2;
            for (int e = wave; e < NTILE + CT / 2; e += NW) {
                if (e >= NTILE) {
                    const int I = 2 * (e - NTILE);
#pragma unroll
                    for (int k = 0; k < NC; ++k) *reinterpret_cast<b16x4 *>(&sm.P[k][I * 16 + lr][(I + 1) * 16 + 4 * lg]) = (b16x4){};
                    continue;
                }
                const int I = (e >= 1) + (e >= 3) + (e >= 6), J = e - I * (I + 1) / 2;
                f32x4 p = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < DC / 32; ++s) {
                    b16x8 x[NP], y[NP];
#pragma unroll
                    for (int k = 0; k < NP; ++k) {
                        x[k] = *reinterpret_cast<const b16x8 *>(&sm.X[k][I * 16 + lr][32 * s + 8 * lg]);
                        y[k] = *reinterpret_cast<const b16x8 *>(&sm.Y[k][J * 16 + lr][32 * s + 8 * lg]);
                    }
                    p = mma<NP, NP>(y, x, p);
                }
                const int i = I * 16 + lr;
                const float gh = sm.Gh[i], gl = sm.Gl[i];
                b16x4 q[NC];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = J * 16 + 4 * lg + r;
                    const float d = fast_exp2((gh - sm.Gh[j]) + (gl - sm.Gl[j]));
                    __bf16 w[NC];
                    split<NC>(j > i ? 0.0f : p[r] * ro.scale_p * d, w);
#pragma unroll
                    for (int k = 0; k < NC; ++k) q[k][r] = w[k];
                }
#pragma unroll
                for (int k = 0; k < NC; ++k) *reinterpret_cast<b16x4 *>(&sm.P[k][i][J * 16 + 4 * lg]) = q[k];
            }
            // ---- O^T = S^T x^T, scaled by 2^{G_i}
#pragma unroll
            for (int I = 0; I < CT; ++I)
#pragma unroll
                for (int n = 0; n < NT; ++n) O[I][n] = (f32x4){0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < DC / 32; ++s) {
                b16x8 st[NT][NC];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        __bf16 w[NC];
                        split<NC>(S[2 * s + j / 4][n][j % 4], w);
#pragma unroll
                        for (int k = 0; k < NC; ++k) st[n][k][j] = w[k];
                    }
#pragma unroll
                for (int I = 0; I < CT; ++I) {
                    b16x8 x[NP];
#pragma unroll
                    for (int k = 0; k < NP; ++k) x[k] = *reinterpret_cast<const b16x8 *>(&sm.X[k][I * 16 + lr][32 * s + 8 * lg]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) O[I][n] = mma<NC, NP>(st[n], x, O[I][n]);
                }
            }
#pragma unroll
            for (int I = 0; I < CT; ++I) {
                const float e = sm.E[I * 16 + lr] * ro.scale_x;
#pragma unroll
                for (int n = 0; n < NT; ++n) O[I][n] *= e;
            }
            __syncthreads();                          // P is whole
        }
#pragma unroll
        for (int t = 0; t < DC / 16; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) S[t][n] *= tot;

        // ---- by 32 tokens: O^T += z^T P^T, S += y^T (2^{G_C - G_j} z_j)
#pragma unroll
        for (int s = 0; s < C / 32; ++s) {
            b16x8 zs[NT][NC];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                b16x8 z[NP];
#pragma unroll
                for (int k = 0; k < NP; ++k)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const b16x4 q = read_tr(&sm.Z[k][32 * s + 8 * lg + 4 * u + lr / 4][zcol0 + 16 * n + 4 * (lr % 4)]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) z[k][4 * u + j] = q[j];
                    }
                if (!STATE_ONLY) {
#pragma unroll
                    for (int I = 2 * s; I < CT; ++I) {
                        b16x8 p[NC];
#pragma unroll
                        for (int k = 0; k < NC; ++k) p[k] = *reinterpret_cast<const b16x8 *>(&sm.P[k][I * 16 + lr][32 * s + 8 * lg]);
                        O[I][n] = mma<NP, NC>(z, p, O[I][n]);
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float v = 0.0f;
#pragma unroll
                    for (int k = NP - 1; k >= 0; --k) v += (float)z[k][j];
                    __bf16 w[NC];
                    split<NC>(v * (sm.R[32 * s + 8 * lg + j] * ro.scale_z), w);
#pragma unroll
                    for (int k = 0; k < NC; ++k) zs[n][k][j] = w[k];
                }
            }
#pragma unroll
            for (int t = 0; t < DC / 16; ++t) {
                b16x8 y[NP];
#pragma unroll
                for (int k = 0; k < NP; ++k)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const b16x4 q = read_tr(&sm.Y[k][32 * s + 8 * lg + 4 * u + lr / 4][32 * (t / 2) + 8 * (lr % 4) + 4 * (t % 2)]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[k][4 * u + j] = q[j];
                    }
#pragma unroll
                for (int n = 0; n < NT; ++n) S[t][n] = mma<NP, NC>(y, zs[n], S[t][n]);
            }
        }

        if (!STATE_ONLY) {
            // ---- the chunk's rows of o
#pragma unroll
            for (int I = 0; I < CT; ++I) {
                const int s = s0 + I * 16 + lr;
                const bool ok = s < len;
                const long long t = ro.reverse ? len - 1 - s : s;
                float dot = 0.0f;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int c = zcol0 + 16 * n + 4 * lg;
                    if (ok && ro.O.p) {
                        const long long at = t * ro.O.st + b * ro.O.sb + h * ro.O.sh + c;
                        if (ro.O.f32) {
                            float *po = reinterpret_cast<float *>(ro.O.p) + at;
                            if (ro.O.vec == 2 && c < dz) *reinterpret_cast<f32x4 *>(po) = O[I][n];
                            else
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    if (c + r < dz) po[r] = O[I][n][r];
                        } else {
                            T *po = reinterpret_cast<T *>(ro.O.p) + at;
                            struct alignas(4 * sizeof(T)) V { T v[4]; } w;
#pragma unroll
                            for (int r = 0; r < 4; ++r) w.v[r] = (T)O[I][n][r];
                            if (ro.O.vec >= (sizeof(T) == 4 ? 2 : 1)) {
                                if (c < dz) *reinterpret_cast<V *>(po) = w;
                            } else
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    if (c + r < dz) po[r] = w.v[r];
                        }
                    }
                    if (ok && ro.dots) {
                        const T *pw = reinterpret_cast<const T *>(ro.W.p) + t * ro.W.st + b * ro.W.sb + (h / ro.W.group) * ro.W.sh + c;
                        if (ro.W.vec >= (sizeof(T) == 4 ? 2 : 1)) {
                            if (c < dz) {
                                struct alignas(4 * sizeof(T)) V { T v[4]; };
                                const V w = *reinterpret_cast<const V *>(pw);
#pragma unroll
                                for (int r = 0; r < 4; ++r) dot += (float)w.v[r] * O[I][n][r];
                            }
                        } else
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (c + r < dz) dot += (float)pw[r] * O[I][n][r];
                    }
                }
                if (ro.dots) {
                    dot += __shfl_xor(dot, 16);
                    dot += __shfl_xor(dot, 32);
                    if (lg == 0) sm.dot[wave][I * 16 + lr] = dot;
                }
            }
        }
    }

    if (STATE_ONLY) {
        f32x4 *so = reinterpret_cast<f32x4 *>(a.states + slot) + (wave * (DC / 16) * NT) * 64 + lane;
#pragma unroll
        for (int t = 0; t < DC / 16; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) so[(t * NT + n) * 64] = S[t][n];
        if (tid == 0) a.decays[(size_t)(ri * BH + bh) * a.nseg + seg] = fast_exp2((float)gsum);
        return;
    }
    if (ro.dots && n_live > 0) {
        __syncthreads();
        flush_dots(first + (n_live - 1) * C);
    }
    // ---- rows behind the sample's length: zeros
    if (ro.O.p) {
        const int r0 = max(first, len);
        for (long long e = tid; e < (long long)(behind - r0) * dz; e += NTHR) {
            const long long at = (r0 + e / dz) * ro.O.st + b * ro.O.sb + h * ro.O.sh + e % dz;
            if (ro.O.f32) reinterpret_cast<float *>(ro.O.p)[at] = 0.0f;
            else reinterpret_cast<T *>(ro.O.p)[at] = (T)0.0f;
        }
    }
    if (ro.s_out && seg == a.nseg - 1) {
        const float more = ro.last_decay && len > 0 ? fast_exp2((float)log2_decay(pg[0])) : 1.0f;
        float *so = ro.s_out + (size_t)bh * dc * dz;
#pragma unroll
        for (int t = 0; t < DC / 16; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = 32 * (t / 2) + 8 * lg + 4 * (t % 2) + i, z = zcol0 + 16 * n + lr;
                    if (c < dc && z < dz) so[c * ro.out_c + z * ro.out_z] = S[t][n][i] * more;
                }
    }
}

template <typename T, int DC, int DZ, int NW>
static int launch_one(const Args &a, bool state_only, hipStream_t stream)
{
    constexpr int C = Kind<T>::NP == 1 ? 64 : 32;     // chunk_tokens()
    const unsigned grid = (unsigned)((size_t)a.B * a.H * a.nseg * a.nroles);
    if (state_only) chunk_kernel<T, DC, DZ, C, NW, true><<<grid, 64 * NW, 0, stream>>>(a);
    else chunk_kernel<T, DC, DZ, C, NW, false><<<grid, 64 * NW, 0, stream>>>(a);
    return launch_status("linear_attention");
}

template <typename T>
int launch_chunks(const Args &a, int DC, int DZ, bool state_only, hipStream_t stream)
{
    // Waves: one 16-column tile of the state each where three planes fill the registers and the LDS leaves room for one
    // workgroup of 128 columns (fp32), two tiles elsewhere.
    constexpr int W128 = Kind<T>::NP == 3 ? 8 : 4;
    if (DC == 32) return launch_one<T, 32, 32, 2>(a, state_only, stream);
    if (DC == 64 && DZ == 64) return launch_one<T, 64, 64, 4>(a, state_only, stream);
    if (DC == 64) return launch_one<T, 64, 128, W128>(a, state_only, stream);
    if (DZ == 64) return launch_one<T, 128, 64, 4>(a, state_only, stream);
    return launch_one<T, 128, 128, W128>(a, state_only, stream);
}

}  // namespace la
}  // namespace dmn
