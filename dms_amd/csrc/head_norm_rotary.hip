// dms_amd/csrc/head_norm_rotary.hip -- RMS norm of every query and key head and its rotation by positions on several
// axes, in one pass, and the gradients of both.
//
//   y = x rsqrt(mean(x^2) + eps) w;   pair (2i, 2i + 1) of y turns by pos[axis(i)] * rate(i); the pairs behind all axes' sections
//   stay as they are.
// Backward, with u = dy turned back:  dw = sum u x r,  dx = r u w - x r^3 mean(x u w),  r = rsqrt(mean(x^2) + eps).
//
// Bound by memory: x is read and y written once (backward: x and dy read, dx written), in 16-byte pieces where the rows
// allow it (bf16, 32 heads of 64 for 163840 tokens: 258 us, 5.2 TB/s, the rate of a copy; fp32, 12 heads of 100 for 128000: 251 us
// and 381 backward, 4.9 TB/s; bf16 and fp16, 32 heads of 64 for 128000: 195 us, 5.4 TB/s, and 320 and 325 backward, 4.9 and 4.8).  A group of 2^lg lanes takes a token and walks its heads, so that cosines and sines are computed once for all of
// them: a lane keeps those of its own E/2 pairs.  The angle is formed in turns and in 64 bits (a position of 2^20 radians
// has lost 4 digits in 32), reduced there, and only the rest of the turn goes on in 32.
#include "common.h"

namespace dmn {
namespace hnr {

constexpr int MAX_PAIRS = 128, MAX_AXES = 4;

struct Table {                        // by value in the launch: the same for every call with the same sections
    double turns[MAX_PAIRS];          // turns for a position step of 1
    int axis[MAX_PAIRS];
    int pairs;                        // pairs that turn
};

struct Rows {                         // element (t, b, h, c) of a tensor at p + t * st + b * sb + h * sh + c
    void *p;
    long long st, sb, sh;
};

struct Args {
    Rows x[2], dy[2], out[2];         // q and k
    const void *w[2];
    int w32;                          // weights in fp32 (else in the type of x)
    const void *pos;
    int pos64;
    long long pt, pb, pa;
    float *partial;                   // (blocks, 2, D) sums of dw, or null
    int heads[2];
    int B, D, lg, nslice, per_slice;
    long long tokens;
    float eps;
    Table table;
};

template <int CTRL>
__device__ __forceinline__ float dpp(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// sum over the 2^lg lanes of a group, the same bits in every lane
__device__ __forceinline__ float group_sum(float v, int lg)
{
    if (lg > 0) v += dpp<0xb1>(v);              // quad_perm 1,0,3,2
    if (lg > 1) v += dpp<0x4e>(v);              // quad_perm 2,3,0,1
    if (lg > 2) v += dpp<0x141>(v);             // row_half_mirror
    if (lg > 3) v += dpp<0x140>(v);             // row_mirror
    if (lg > 4) v += __shfl_xor(v, 16);
    if (lg > 5) v += __shfl_xor(v, 32);
    return v;
}

template <typename T, int E> struct alignas(E * sizeof(T)) Piece { T v[E]; };

// E elements of a row from column c on; VEC: the row's pieces are aligned and whole
template <typename T, int E, bool VEC>
__device__ __forceinline__ void load(const T *row, int c, int D, float (&x)[E])
{
    if (VEC) {
        const Piece<T, E> p = *reinterpret_cast<const Piece<T, E> *>(row + c);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = (float)p.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = c + i < D ? (float)row[c + i] : 0.0f;
    }
}

template <typename T, int E, bool VEC>
__device__ __forceinline__ void store(T *row, int c, int D, const float (&x)[E])
{
    if (VEC) {
        Piece<T, E> p;
#pragma unroll
        for (int i = 0; i < E; ++i) p.v[i] = (T)x[i];
        *reinterpret_cast<Piece<T, E> *>(row + c) = p;
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (c + i < D) row[c + i] = (T)x[i];
    }
}

template <typename T, int E>
__device__ __forceinline__ void load_weight(const void *w, int w32, int c, int D, float (&x)[E])
{
#pragma unroll
    for (int i = 0; i < E; ++i) {
        x[i] = 1.0f;
        if (w && c + i < D) x[i] = w32 ? static_cast<const float *>(w)[c + i] : (float)static_cast<const T *>(w)[c + i];
    }
}

// cosine and sine of the lane's pairs at token (t, b)
template <int E>
__device__ __forceinline__ void angles(const Args &a, long long t, long long b, int c, float (&co)[E / 2], float (&si)[E / 2])
{
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
        const int pair = c / 2 + i;
        co[i] = 1.0f;
        si[i] = 0.0f;
        if (pair < a.table.pairs) {
            const long long at = t * a.pt + b * a.pb + a.table.axis[pair] * a.pa;
            const long long pos = a.pos64 ? static_cast<const long long *>(a.pos)[at] : (long long)static_cast<const int *>(a.pos)[at];
            double n = (double)pos * a.table.turns[pair];
            n -= rint(n);
            sincospif(2.0f * (float)n, &si[i], &co[i]);
        }
    }
}

// gridDim.y slices of the heads where there are few tokens
template <typename T, int E, bool VEC>
__global__ void __launch_bounds__(256) forward_kernel(const Args a)
{
    const int group = threadIdx.x >> a.lg, c = (threadIdx.x & ((1 << a.lg) - 1)) * E;
    const long long token = (long long)blockIdx.x * (256 >> a.lg) + group;
    if (token >= a.tokens) return;                        // whole groups leave: no lane of the others needs them
    const long long t = token / a.B, b = token % a.B;
    const bool ok = c < a.D;
    float co[E / 2], si[E / 2];
    angles<E>(a, t, b, c, co, si);
    const int all = a.heads[0] + a.heads[1], h0 = blockIdx.y * a.per_slice, h1 = min(all, h0 + a.per_slice);
    const float inv = 1.0f / (float)a.D;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const int lo = m ? max(h0 - a.heads[0], 0) : h0, hi = m ? h1 - a.heads[0] : min(h1, a.heads[0]);
        if (lo >= hi) continue;
        float w[E];
        load_weight<T, E>(a.w[m], a.w32, c, a.D, w);
        const T *px = static_cast<const T *>(a.x[m].p) + t * a.x[m].st + b * a.x[m].sb;
        T *py = static_cast<T *>(a.out[m].p) + t * a.out[m].st + b * a.out[m].sb;
#pragma unroll 4
        for (int h = lo; h < hi; ++h) {
            float x[E];
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = 0.0f;
            if (ok) load<T, E, VEC>(px + h * a.x[m].sh, c, a.D, x);
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < E; ++i) ss += x[i] * x[i];
            const float r = rsqrtf(group_sum(ss, a.lg) * inv + a.eps);
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                const float p = x[i] * r * w[i], q = x[i + 1] * r * w[i + 1];
                x[i] = p * co[i / 2] - q * si[i / 2];
                x[i + 1] = p * si[i / 2] + q * co[i / 2];
            }
            if (ok) store<T, E, VEC>(py + h * a.out[m].sh, c, a.D, x);
        }
    }
}

// A group walks tokens gridDim.x * groups apart and keeps its sums of dw; they are joined over the workgroup in LDS, over
// the workgroups by sum_kernel, always in the same order.
template <typename T, int E, bool VEC>
__global__ void __launch_bounds__(256) backward_kernel(const Args a)
{
    __shared__ float sh[256 * E];
    const int group = threadIdx.x >> a.lg, groups = 256 >> a.lg, c = (threadIdx.x & ((1 << a.lg) - 1)) * E;
    const bool ok = c < a.D;
    const float inv = 1.0f / (float)a.D;
    float w[2][E], dw[2][E];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        load_weight<T, E>(a.w[m], a.w32, c, a.D, w[m]);
#pragma unroll
        for (int i = 0; i < E; ++i) dw[m][i] = 0.0f;
    }
    const int all = a.heads[0] + a.heads[1], h0 = blockIdx.y * a.per_slice, h1 = min(all, h0 + a.per_slice);
    for (long long token = (long long)blockIdx.x * groups + group; token < a.tokens; token += (long long)gridDim.x * groups) {
        const long long t = token / a.B, b = token % a.B;
        float co[E / 2], si[E / 2];
        angles<E>(a, t, b, c, co, si);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int lo = m ? max(h0 - a.heads[0], 0) : h0, hi = m ? h1 - a.heads[0] : min(h1, a.heads[0]);
            const T *px = static_cast<const T *>(a.x[m].p) + t * a.x[m].st + b * a.x[m].sb;
            const T *pd = static_cast<const T *>(a.dy[m].p) + t * a.dy[m].st + b * a.dy[m].sb;
            T *po = static_cast<T *>(a.out[m].p) + t * a.out[m].st + b * a.out[m].sb;
#pragma unroll 2
            for (int h = lo; h < hi; ++h) {
                float x[E], u[E];
#pragma unroll
                for (int i = 0; i < E; ++i) x[i] = u[i] = 0.0f;
                if (ok) {
                    load<T, E, VEC>(px + h * a.x[m].sh, c, a.D, x);
                    load<T, E, VEC>(pd + h * a.dy[m].sh, c, a.D, u);
                }
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < E; ++i) ss += x[i] * x[i];
                const float r = rsqrtf(group_sum(ss, a.lg) * inv + a.eps);
                float xu = 0.0f;
#pragma unroll
                for (int i = 0; i < E; i += 2) {
                    const float p = u[i] * co[i / 2] + u[i + 1] * si[i / 2], q = u[i + 1] * co[i / 2] - u[i] * si[i / 2];
                    x[i] *= r;                            // from here x is the normalised row
                    x[i + 1] *= r;
                    dw[m][i] += p * x[i];
                    dw[m][i + 1] += q * x[i + 1];
                    u[i] = p * w[m][i];
                    u[i + 1] = q * w[m][i + 1];
                    xu += x[i] * u[i] + x[i + 1] * u[i + 1];
                }
                const float mean = group_sum(xu, a.lg) * inv;
#pragma unroll
                for (int i = 0; i < E; ++i) u[i] = r * (u[i] - x[i] * mean);
                if (ok) store<T, E, VEC>(po + h * a.out[m].sh, c, a.D, u);
            }
        }
    }
    if (!a.partial) return;
    const int cols = (1 << a.lg) * E;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < E; ++i) sh[group * cols + c + i] = dw[m][i];
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += 256) {
            float s = 0.0f;
            for (int g = 0; g < groups; ++g) s += sh[g * cols + d];
            a.partial[((size_t)(blockIdx.y * gridDim.x + blockIdx.x) * 2 + m) * a.D + d] = s;
        }
    }
}

// dw (2, D) = sum over the blocks, in block order in 64 bits: 8 threads a column, then their 8 sums
template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(const float *partial, void *dwq, void *dwk, int w32, int blocks, int D)
{
    __shared__ double sh[256];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    double s = 0.0;
    if (col < 2 * D) {
        const int n = (blocks + 7) / 8, lo = part * n, hi = min(blocks, lo + n);
#pragma unroll 8
        for (int i = lo; i < hi; ++i) s += (double)partial[(size_t)i * 2 * D + col];
    }
    sh[threadIdx.x] = s;
    __syncthreads();
    if (part == 0 && col < 2 * D) {
        for (int i = 1; i < 8; ++i) s += sh[i * 32 + threadIdx.x];
        void *out = col < D ? dwq : dwk;
        const int d = col < D ? col : col - D;
        if (out) {
            if (w32) static_cast<float *>(out)[d] = (float)s;
            else static_cast<T *>(out)[d] = (T)(float)s;
        }
    }
}

// ------------------------------------------------------------------------------------------------ host side
static int elem(int dtype) { return dtype == 0 ? 4 : 2; }

static Rows rows(const void *p, int T, int B, int H, const long long *s)
{
    Rows r;
    r.p = const_cast<void *>(p);
    r.st = T > 1 ? s[0] : 0;
    r.sb = B > 1 ? s[1] : 0;
    r.sh = H > 1 ? s[2] : 0;
    return r;
}

static Rows dense(void *p, int T, int B, int H, int D)
{
    const long long s[3] = {(long long)B * H * D, (long long)H * D, D};
    return rows(p, T, B, H, s);
}

static bool pieces(const Rows &r, int es, int D, int bytes)
{
    return (((unsigned long long)(size_t)r.p | (unsigned long long)(r.st * es) | (unsigned long long)(r.sb * es) |
             (unsigned long long)(r.sh * es) | (unsigned long long)D * es) % bytes) == 0;
}

constexpr int MAX_BLOCKS = 4 * NUM_CU;      // of the backward: its dw sums are joined over this many at most

struct Shape {
    int E, vec, lg;
};

// 16 bytes a lane where all rows allow it, else 4 elements (8-byte pieces of 16-bit rows, or one at a time)
static Shape shape(const Args &a, int dtype, bool backward)
{
    const int es = elem(dtype);
    const auto all = [&](int bytes) {
        for (int m = 0; m < 2; ++m)
            if (a.heads[m] && (!pieces(a.x[m], es, a.D, bytes) || !pieces(a.out[m], es, a.D, bytes) ||
                               (backward && !pieces(a.dy[m], es, a.D, bytes)))) return false;
        return true;
    };
    Shape s;
    s.E = 16 / es;
    s.vec = all(16);
    if (!s.vec) {
        s.E = 4;
        s.vec = all(4 * es);
    }
    s.lg = 0;
    while ((s.E << s.lg) < a.D) ++s.lg;
    return s;
}

template <typename T, int E>
static void launch(const Args &a, bool vec, bool backward, dim3 grid, hipStream_t st)
{
    if (backward) {
        if (vec) backward_kernel<T, E, true><<<grid, 256, 0, st>>>(a);
        else backward_kernel<T, E, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (vec) forward_kernel<T, E, true><<<grid, 256, 0, st>>>(a);
        else forward_kernel<T, E, false><<<grid, 256, 0, st>>>(a);
    }
}

static int run(const char *who, int dtype, Args &a, bool backward, hipStream_t st)
{
    const Shape s = shape(a, dtype, backward);
    a.lg = s.lg;
    const int groups = 256 >> s.lg, all = a.heads[0] + a.heads[1];
    long long blocks = (a.tokens + groups - 1) / groups;
    if (backward && blocks > MAX_BLOCKS) blocks = MAX_BLOCKS;
    if (blocks > 0xffffffLL) return fail(-6, "%s: %lld tokens exceed one grid", who, a.tokens);
    // few tokens: the heads go over the grid as well, at the price of the angles once more for each slice
    a.nslice = 1;
    while (a.nslice < all && blocks * a.nslice < 2 * NUM_CU) a.nslice *= 2;
    a.per_slice = (all + a.nslice - 1) / a.nslice;
    a.nslice = (all + a.per_slice - 1) / a.per_slice;
    const dim3 grid((unsigned)blocks, (unsigned)a.nslice);
    if (dtype == 0) launch<float, 4>(a, s.vec, backward, grid, st);
    else if (dtype == 1) s.E == 8 ? launch<__bf16, 8>(a, s.vec, backward, grid, st) : launch<__bf16, 4>(a, s.vec, backward, grid, st);
    else s.E == 8 ? launch<_Float16, 8>(a, s.vec, backward, grid, st) : launch<_Float16, 4>(a, s.vec, backward, grid, st);
    return launch_status(who);
}

static int check(const char *who, int dtype, int T, int B, int Hq, int Hk, int D, const int *sections, int axes, const double *rates)
{
    if (dtype < 0 || dtype > 2) return fail(-2, "%s: dtype must be 0 (fp32), 1 (bf16) or 2 (fp16), got %d", who, dtype);
    if (T < 0 || B < 0 || Hq < 1 || Hk < 0) return fail(-3, "%s: bad sizes T=%d B=%d Hq=%d Hk=%d", who, T, B, Hq, Hk);
    if (D < 1 || D > 256) return fail(-5, "%s: head widths must be 1 .. 256, got %d", who, D);
    if (axes < 0 || axes > MAX_AXES || (axes > 0 && !sections)) return fail(-4, "%s: 0 .. %d axes, got %d", who, MAX_AXES, axes);
    int sum = 0;
    for (int i = 0; i < axes; ++i) {
        if (sections[i] < 0 || sections[i] > MAX_PAIRS) return fail(-4, "%s: bad section of %d pairs", who, sections[i]);
        sum += sections[i];
    }
    if (sum > D / 2) return fail(-4, "%s: %d pairs turn, a head of width %d has %d", who, sum, D, D / 2);
    if (sum > 0 && !rates) return fail(-1, "%s: null pointer", who);
    return 0;
}

static void fill(Args &a, const void *q, const void *k, const void *wq, const void *wk, int w32, const void *pos, int pos64, const int *sections,
                 int axes, const double *rates, float eps, const long long *s, int T, int B, int Hq, int Hk, int D)
{
    a.x[0] = rows(q, T, B, Hq, s);
    a.x[1] = rows(k, T, B, Hk, s + 3);
    a.dy[0] = a.dy[1] = a.x[0];
    a.w[0] = wq;
    a.w[1] = wk;
    a.w32 = w32;
    a.pos = pos;
    a.pos64 = pos64;
    a.pt = T > 1 ? s[6] : 0;
    a.pb = B > 1 ? s[7] : 0;
    a.pa = s[8];
    a.partial = nullptr;
    a.heads[0] = Hq;
    a.heads[1] = Hk;
    a.B = B;
    a.D = D;
    a.tokens = (long long)T * B;
    a.eps = eps;
    a.table.pairs = 0;
    for (int i = 0; i < axes; ++i)
        for (int j = 0; j < sections[i]; ++j) {
            a.table.turns[a.table.pairs] = rates[a.table.pairs] * 0.15915494309189533576888376337251;      // 1 / 2 pi
            a.table.axis[a.table.pairs++] = i;
        }
}

}  // namespace hnr
}  // namespace dmn

using namespace dmn;
using namespace dmn::hnr;

extern "C" int dmn_head_norm_rotary_fwd(int dtype, const void *q, const void *k, const void *wq, const void *wk, int w32, const void *positions,
                                        int positions64, const int *sections, int axes, const double *rates, float eps, void *yq, void *yk,
                                        const long long *strides, int T, int B, int Hq, int Hk, int D, void *stream)
{
    const char *who = "dmn_head_norm_rotary_fwd";
    const int rc = check(who, dtype, T, B, Hq, Hk, D, sections, axes, rates);
    if (rc) return rc;
    if (!strides || (T > 0 && B > 0 && (!q || !yq || (Hk && (!k || !yk)) || (axes > 0 && !positions)))) return fail(-1, "%s: null pointer", who);
    if ((long long)T * B == 0) return 0;
    Args a;
    fill(a, q, k, wq, wk, w32, positions, positions64, sections, axes, rates, eps, strides, T, B, Hq, Hk, D);
    a.out[0] = dense(yq, T, B, Hq, D);
    a.out[1] = dense(yk, T, B, Hk, D);
    return run(who, dtype, a, false, (hipStream_t)stream);
}

extern "C" int dmn_head_norm_rotary_workspace_floats(int Hq, int Hk, int D)
{
    if (Hq < 1 || Hk < 0 || D < 1 || D > 256) return -1;
    return MAX_BLOCKS * 2 * D;            // slices are doubled below 2 * NUM_CU blocks: never more than 4 * NUM_CU either
}

extern "C" int dmn_head_norm_rotary_bwd(int dtype, const void *q, const void *k, const void *wq, const void *wk, int w32, const void *positions,
                                        int positions64, const int *sections, int axes, const double *rates, float eps, const void *grad_yq,
                                        const void *grad_yk, void *grad_q, void *grad_k, void *grad_wq, void *grad_wk, const long long *strides,
                                        float *workspace, int T, int B, int Hq, int Hk, int D, void *stream)
{
    const char *who = "dmn_head_norm_rotary_bwd";
    int rc = check(who, dtype, T, B, Hq, Hk, D, sections, axes, rates);
    if (rc) return rc;
    if (!strides || (T > 0 && B > 0 && (!q || !grad_yq || !grad_q || (Hk && (!k || !grad_yk || !grad_k)) || (axes > 0 && !positions))))
        return fail(-1, "%s: null pointer", who);
    const bool weights = grad_wq || grad_wk;
    if (weights && !workspace) return fail(-7, "%s: needs a workspace", who);
    hipStream_t st = (hipStream_t)stream;
    Args a;
    a.nslice = 0;
    long long blocks = 0;
    if ((long long)T * B > 0) {
        fill(a, q, k, wq, wk, w32, positions, positions64, sections, axes, rates, eps, strides, T, B, Hq, Hk, D);
        a.dy[0] = rows(grad_yq, T, B, Hq, strides + 9);
        a.dy[1] = rows(grad_yk, T, B, Hk, strides + 12);
        a.out[0] = dense(grad_q, T, B, Hq, D);
        a.out[1] = dense(grad_k, T, B, Hk, D);
        a.partial = weights ? workspace : nullptr;
        rc = run(who, dtype, a, true, st);
        if (rc) return rc;
        blocks = (a.tokens + (256 >> a.lg) - 1) / (256 >> a.lg);
        if (blocks > MAX_BLOCKS) blocks = MAX_BLOCKS;
        blocks *= a.nslice;
    }
    if (!weights) return 0;
    const unsigned grid = (2 * D + 31) / 32;
    if (dtype == 0) sum_kernel<float><<<grid, 256, 0, st>>>(workspace, grad_wq, grad_wk, w32, (int)blocks, D);
    else if (dtype == 1) sum_kernel<__bf16><<<grid, 256, 0, st>>>(workspace, grad_wq, grad_wk, w32, (int)blocks, D);
    else sum_kernel<_Float16><<<grid, 256, 0, st>>>(workspace, grad_wq, grad_wk, w32, (int)blocks, D);
    return launch_status(who);
}
