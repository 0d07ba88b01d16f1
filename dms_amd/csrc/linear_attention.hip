// dms_amd/csrc/linear_attention.hip -- entry points of linear attention with a decay for each head, the small kernels
// round the chunk kernels (linear_attention.inl), and the single-token step.
#include "linear_attention.h"

namespace dmn {
namespace la {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

// states[seg] = state after segment seg, from what each segment added: one thread for 4 elements of the state, in
// segment order (at most NUM_CU), so the same bits every time.  8 segments are loaded at a time, as what this costs is the
// loads' latency: 16 heads of 64 x 64 in 16 segments 4.4 us, one head of 32768 tokens in 256 segments 27 us of 45 in all.
__global__ void __launch_bounds__(64) combine_kernel(float *states, const double *decays, int nseg, int n4, long long total)
{
    const long long e = (long long)blockIdx.x * 64 + threadIdx.x;
    if (e >= total) return;
    const long long row = e / n4;
    f32x4 *p = reinterpret_cast<f32x4 *>(states) + row * nseg * n4 + e % n4;
    const double *d = decays + row * nseg;
    f64x4 s = __builtin_convertvector(p[0], f64x4);        // rounded where it is kept, not where it goes on
    for (int i = 1; i < nseg - 1; i += 8) {
        f32x4 add[8];
        double decay[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int at = i + k < nseg - 1 ? i + k : nseg - 2;
            add[k] = p[(long long)at * n4];
            decay[k] = d[at];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + k < nseg - 1) {
                s = s * decay[k] + __builtin_convertvector(add[k], f64x4);
                p[(long long)(i + k) * n4] = __builtin_convertvector(s, f32x4);
            }
    }
}

// out (rows, heads, d) = sum over the group of in (rows, heads * group, d), in head order
template <typename T>
__global__ void __launch_bounds__(256) group_sum_kernel(const float *in, T *out, int heads, int group, int d, long long total)
{
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
        const long long row = e / d;                      // (token, sample, head)
        const float *p = in + row * group * d + e % d;
        float s = 0.0f;
        for (int u = 0; u < group; ++u) s += p[(long long)u * d];
        out[e] = (T)s;
    }
}

template <int N>
__device__ __forceinline__ double block_sum(double v, double *sh)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < N / 64; ++w) s += sh[w];
    return s;
}

// Gradient of the log decays.  What flows over the border before token t -- dg_t = <a_t S_{t-1}, dS_t> -- is what came in before
// an earlier token s less what the tokens between took out of the keys' side over the queries':
//   dg_t = dg_s - sum_{s <= i < t} (q_i . dq_i - k_i . dk_i)
// The dots are right to fp32, and their running sum walks away from the truth with the root of the distance.  So dg is known
// directly at every ANCHOR-th token, from the two states that meet there, at the first (<S_0, dS_0>) and behind the last
// (<S_T, dS_T>; not of up to 64 tokens, which have no way to walk: 512 heads of 125 x 125 would pay 20 us for 20): a sum starts at each and what it
// misses at the next is spread over the way (2046 tokens: an error of 2.2e-6 of the norm without, 4.4e-7 with).
//
// flow[bh][i] = <S, dS> between the tokens before and from the anchor i + 1 on, n4 fours of either state in the same order.  Bound by
// reading them: 41 us, 5.7 TB/s, for 1024 heads of 64 x 64 and 2000 tokens; every 512th token would halve that, and leave 1.4 times
// the error.
__global__ void __launch_bounds__(256) meet_kernel(const f32x4 *before, const f32x4 *behind, double *flow, int n4)
{
    __shared__ double sh[4];
    double sum = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n4; i += 256) {
        const f32x4 a = before[(size_t)blockIdx.x * n4 + i], b = behind[(size_t)blockIdx.x * n4 + i];
#pragma unroll
        for (int k = 0; k < 4; ++k) sum += (double)a[k] * (double)b[k];
    }
    sum = block_sum<256>(sum, sh);
    if (threadIdx.x == 0) flow[blockIdx.x] = sum;
}

// Tokens from which on <S_T, dS_T> is taken: 256 heads of 128 x 128 in fp32, 65 tokens: 192 in place of 184 us, the error 4.1e-7 ->
// 2.5e-7 of the norm, of the last 8 tokens 6.6e-7 -> 2.0e-7; 256 tokens: 262 and 245 us, 7.6e-7 -> 4.4e-7 and 1.5e-6 -> 2.1e-7.
constexpr int END_FROM = 65;

// workgroups of a (sample, head) in the scan below
__host__ __device__ static inline int stretches(int T) { return (T + 4 * ANCHOR - 1) / (4 * ANCHOR); }

// A wave for each stretch between anchors, four a workgroup, in 64 bits; the result takes the dots' place, or its sum goes to
// `part`: g and dg have the heads together, and 4 bytes of every line would be written from here (44 us for 1024 heads of 2000
// tokens; this takes 15, the turn below 17).
__global__ void __launch_bounds__(256)
decay_scan_kernel(float *dots_q, const float *dots_k, const double *flow, const float *s0, const float *ds0, const float *s_end, const float *ds_end,
                  const float *g, long long gt, long long gb, long long gh, const void *lengths, int lengths64, double *part, int T, int B, int H, int n)
{
    constexpr int N = ANCHOR / 64;                         // tokens a lane
    __shared__ double sh[4];
    const int bh = blockIdx.x % (B * H), at = blockIdx.x / (B * H), b = bh / H, h = bh % H, tid = threadIdx.x, lane = tid & 63;
    const int n_anchor = anchors(T), len = valid_length(lengths, lengths64, b, T);
    const float *pg = g + b * gb + h * gh;
    const auto meet = [&](const float *x, const float *y) {
        double v = 0.0;
#pragma unroll 8
        for (int i = tid; i < n; i += 256) v += (double)x[(size_t)bh * n + i] * (double)y[(size_t)bh * n + i];
        v = block_sum<256>(v, sh);
        __syncthreads();
        return v;
    };
    const double first = at == 0 && s0 ? meet(s0, ds0) : 0.0;
    const double end = at == (len - 1) / (4 * ANCHOR) && s_end ? meet(s_end, ds_end) : 0.0;
    const int a = 4 * at + (tid >> 6), t_a = a * ANCHOR;   // this stretch begins at anchor a
    const auto known = [&](int i) {                        // dg at anchor i, or behind the last token
        if (i * ANCHOR >= len) return end;
        return i == 0 ? first : flow[(size_t)bh * n_anchor + i - 1] * (double)fast_exp2((float)log2_decay(pg[(long long)i * ANCHOR * gt]));
    };
    double sum = 0.0;
    if (t_a < T) {
        float *pq = dots_q + (size_t)bh * T;
        const float *pk = dots_k + (size_t)bh * T;
        double d[N], mine = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int t = t_a + lane * N + i;
            d[i] = t < len ? (double)pq[t] - (double)pk[t] : 0.0;
            mine += d[i];
        }
        const double upto = lane_sums(mine), from = t_a < len ? known(a) : 0.0;
        const bool tied = t_a < len && (s_end || !ds_end || t_a + ANCHOR < len);
        const double off = tied ? (from - __shfl(upto, 63) - known(a + 1)) / (double)min(ANCHOR, len - t_a) : 0.0;
        double v = from - (upto - mine);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int t = t_a + lane * N + i;
            if (t < T) {
                const double x = t < len ? v - off * (double)(t - t_a) : 0.0;
                if (part) sum += x;
                else pq[t] = (float)x;
            }
            v -= d[i];
        }
    }
    if (part) {
        sum = block_sum<256>(sum, sh);
        if (tid == 0) part[(size_t)bh * stretches(T) + at] = log2_decay(pg[0]) < -149.0 ? 0.0 : sum;
    }
}

// dg (T, B*H) from its scan (B*H, T), 64 x 64 at a time; a decay of zero has no gradient
__global__ void __launch_bounds__(256)
decay_turn_kernel(const float *scan, const float *g, long long gt, long long gb, long long gh, float *out, int T, int BH, int H)
{
    __shared__ float tile[64][65];
    const int t0 = blockIdx.x * 64, x0 = blockIdx.y * 64, lane = threadIdx.x & 63, row = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int x = x0 + row + 4 * i, t = t0 + lane;
        if (x < BH && t < T) tile[row + 4 * i][lane] = scan[(size_t)x * T + t];
    }
    __syncthreads();
    const int x = x0 + lane;
    if (x >= BH) return;
    const float *pg = g + (x / H) * gb + (x % H) * gh;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int t = t0 + row + 4 * i;
        if (t < T) out[(size_t)t * BH + x] = log2_decay(pg[(long long)t * gt]) < -149.0 ? 0.0f : tile[lane][row + 4 * i];
    }
}

// one decay for each head: its gradient is the sum over samples and stretches, a wave for each head, always in the same order
__global__ void __launch_bounds__(64) decay_grad_heads_kernel(const double *part, float *out, int B, int H, int stretches)
{
    double s = 0.0;
    for (int e = threadIdx.x; e < B * stretches; e += 64) s += part[((size_t)(e / stretches) * H + blockIdx.x) * stretches + e % stretches];
    s = lane_sums(s);
    if (threadIdx.x == 63) out[blockIdx.x] = (float)s;
}

// One token: S = a S + k^T v in place, o = scale q S.  Bound by reading and writing the state once (256 streams of 16 heads of
// 128 x 128: 537 MB in 99 us, 5.4 TB/s; 8 heads of 125 x 125: 5 us, a launch).  A workgroup takes
// a head, or a slice of its columns where there are few heads (a row of S then still comes in whole 64-byte pieces);
// V columns a thread (4 where every row is 16-byte aligned), rows over the threads, their partial o joined in LDS in
// row order.
template <typename T, int V>
__global__ void __launch_bounds__(256)
step_kernel(const T *q, const T *k, const T *v, const float *g, float *state, T *o, long long qb, long long qh, long long kb, long long kh,
            long long vb, long long vh, long long gb, long long gh, long long sb, int H, int gq, int gk, int gv, int dk, int dv, int zb,
            int lz, float scale)
{
    __shared__ float sq[128], sk[128], part[256 * V];
    const int bh = blockIdx.x, b = bh / H, h = bh % H, tid = threadIdx.x;
    if (tid < dk) {
        sq[tid] = (float)q[b * qb + (h / gq) * qh + tid];
        sk[tid] = (float)k[b * kb + (h / gk) * kh + tid];
    }
    const float a = fast_exp2((float)log2_decay(g[b * gb + h * gh]));
    const int z_lanes = 1 << lz, rows = 256 >> lz, zi = tid & (z_lanes - 1), ci = tid >> lz;
    const int z = blockIdx.y * zb + zi * V;
    const bool ok = zi * V < zb && z < dv;
    float vv[V], acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        vv[i] = ok ? (float)v[b * vb + (h / gv) * vh + z + i] : 0.0f;
        acc[i] = 0.0f;
    }
    __syncthreads();
    if (ok) {
        struct alignas(4 * V) Vec { float x[V]; };
        float *p = state + b * sb + (long long)h * dk * dv + z;
#pragma unroll 8
        for (int c = ci; c < dk; c += rows) {
            Vec s = *reinterpret_cast<const Vec *>(p + (long long)c * dv);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s.x[i] = s.x[i] * a + sk[c] * vv[i];
                acc[i] += sq[c] * s.x[i];
            }
            *reinterpret_cast<Vec *>(p + (long long)c * dv) = s;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) part[(ci * z_lanes + zi) * V + i] = acc[i];
    __syncthreads();
    const int cols = min(zb, dv - (int)blockIdx.y * zb);
    for (int c = tid; c < cols; c += 256) {
        float s = 0.0f;
        for (int r = 0; r < rows; ++r) s += part[r * z_lanes * V + c];
        o[(long long)bh * dv + blockIdx.y * zb + c] = (T)(s * scale);
    }
}

// ------------------------------------------------------------------------------------------------ host side
struct Plan {
    int DC, DZ, nchunks, nseg, seg_chunks;
};

static int padded(int d) { return d <= 32 ? 32 : (d <= 64 ? 64 : 128); }

static void pad_pair(int dc, int dz, int *DC, int *DZ)
{
    *DC = padded(dc);
    *DZ = padded(dz);
    if (*DC != *DZ) {                                      // 32 goes with 32 alone
        if (*DC == 32) *DC = 64;
        if (*DZ == 32) *DZ = 64;
    }
}

// Segments: a sequence is cut where the (sample, head) pairs alone leave compute units without a workgroup, into as many as give
// each one, at the cost of reading y and z once more for the states between segments.  16 heads of 5120 tokens: 33.7 us with
// 16 segments, 34.0 with 32, 37.8 with 48; 32 heads of 1999 tokens with their backward: 256 us with 8, 262 with 16, 287 with 24.
// From 129 pairs on that is two segments, which pays where two workgroups fit a compute unit (64 x 64: 130 ragged fp32 sequences of
// up to 2000 tokens 138 us, uncut 153; 250 of 2000: 191 and 196) and where few ragged ones leave units idle (128 x 128, 130 ragged, fp32: 227 us,
// uncut 278), but not for 128 x 128 with more or full sequences, whose workgroups then take two turns (130 of 2000: 370 us, uncut 304;
// 250 ragged: 373 and 302).
static void plan_segments(int dtype, int T, long long passes, int *nseg, int *seg_chunks)
{
    const int C = chunk_tokens(dtype), nchunks = (T + C - 1) / C;
    long long want = passes > 0 && passes < NUM_CU ? (NUM_CU + passes - 1) / passes : 1;
    const int most = nchunks / 2 > 1 ? nchunks / 2 : 1;    // two chunks at least: a shorter segment costs more than it hides
    if (want > most) want = most;
    *seg_chunks = nchunks ? (nchunks + (int)want - 1) / (int)want : 1;
    *nseg = nchunks ? (nchunks + *seg_chunks - 1) / *seg_chunks : 1;
}

// a chunk of tokens has to lie within the 4 GiB that a buffer access reaches
static bool reaches(const long long *s, int T, int tensors)
{
    if (T <= 1) return true;
    for (int i = 0; i < tensors; ++i)
        if (s[3 * i] < 0 || s[3 * i] > (1LL << 24) + (1 << 20)) return false;
    return true;
}

static Tensor tensor(const void *p, int dtype, int T, int B, int heads, int H, int d, const long long *s)
{
    Tensor t;
    t.p = static_cast<char *>(const_cast<void *>(p));
    t.st = T > 1 ? s[0] : 0;
    t.sb = B > 1 ? s[1] : 0;
    t.sh = heads > 1 ? s[2] : 0;
    t.d = d;
    t.group = H / heads;
    t.f32 = 0;
    const unsigned long long es = (unsigned long long)elem_size(dtype);
    const unsigned long long bits = (unsigned long long)(size_t)p | (unsigned long long)t.st * es | (unsigned long long)t.sb * es |
                                    (unsigned long long)t.sh * es | (unsigned long long)d * es;
    t.vec = bits % 16 == 0 ? 2 : (bits % 8 == 0 ? 1 : 0);
    return t;
}

static Tensor dense(void *p, int dtype, int T, int B, int H, int d)
{
    const long long s[3] = {(long long)B * H * d, (long long)H * d, d};
    return tensor(p, dtype, T, B, H, H, d, s);
}

static long long up4(long long n) { return (n + 3) & ~3LL; }

static int launch(int dtype, const Args &a, int DC, int DZ, int kind, hipStream_t stream)
{
    if (dtype == DTYPE_BF16) return launch_chunks<__bf16>(a, DC, DZ, kind, stream);
    if (dtype == DTYPE_F16) return launch_chunks<_Float16>(a, DC, DZ, kind, stream);
    return launch_chunks<float>(a, DC, DZ, kind, stream);
}

// all passes of `a` (same DC, DZ): states between segments first where there are several
static int run_passes(int dtype, Args &a, int DC, int DZ, int kind, float *ws, hipStream_t stream)
{
    if (a.nseg > 1) {
        const long long rows = (long long)a.nroles * a.B * a.H;
        a.states = ws;
        a.decays = reinterpret_cast<double *>(ws + rows * a.nseg * DC * DZ);
        int rc = launch(dtype, a, DC, DZ, kind | STATES, stream);
        if (rc) return rc;
        if (a.nseg > 2) {
            const int n4 = DC * DZ / 4;
            const long long total = rows * n4;
            combine_kernel<<<(unsigned)((total + 63) / 64), 64, 0, stream>>>(a.states, a.decays, a.nseg, n4, total);
            rc = launch_status("linear_attention combine");
            if (rc) return rc;
        }
    }
    return launch(dtype, a, DC, DZ, kind, stream);
}

static long long passes_floats(int nroles, long long BH, int nseg, int DC, int DZ)
{
    return nseg > 1 ? up4((long long)nroles * BH * nseg * DC * DZ) + up4(2LL * nroles * BH * nseg) : 0;
}

static int check(const char *who, int dtype, int T, int B, int H, int Hq, int Hk, int Hv, int dk, int dv)
{
    if (dtype < 0 || dtype > 2) return fail(-2, "%s: dtype must be 0 (fp32), 1 (bf16) or 2 (fp16), got %d", who, dtype);
    if (T < 0 || B < 0 || H < 1 || Hq < 1 || Hk < 1 || Hv < 1)
        return fail(-3, "%s: bad sizes T=%d B=%d H=%d Hq=%d Hk=%d Hv=%d", who, T, B, H, Hq, Hk, Hv);
    if (H % Hq || H % Hk || H % Hv) return fail(-4, "%s: the %d heads of the state must be a multiple of Hq=%d, Hk=%d and Hv=%d", who, H, Hq, Hk, Hv);
    if (dk < 1 || dk > 128 || dv < 1 || dv > 128) return fail(-5, "%s: head widths must be 1 .. 128, got dk=%d dv=%d", who, dk, dv);
    if ((long long)B * H > (1 << 17)) return fail(-6, "%s: B * H = %lld exceeds 2^17", who, (long long)B * H);
    if (T > 1 << 29 || (long long)T * B * H > 0xffffffffLL)   // threads of a grid
        return fail(-6, "%s: T = %d exceeds 2^29, or T * B * H = %lld 2^32", who, T, (long long)T * B * H);
    return 0;
}

static void fill_common(Args &a, const float *g, const long long *gs, const void *lengths, int lengths64, int T, int B, int H)
{
    a.g = g;
    a.gt = gs[0];
    a.gb = gs[1];
    a.gh = gs[2];
    a.lengths = lengths;
    a.lengths64 = lengths64;
    a.T = T;
    a.B = B;
    a.H = H;
    a.states = nullptr;
    a.decays = nullptr;
}

// the backward's passes: where each one's piece of the workspace begins; decays: their gradient is wanted
struct BwdPlan {
    int DK, DV;
    long long passes, keep[2], flow, dots, dq, dk, dv, ds0, end, part, total;
};

static BwdPlan plan_bwd(int dtype, bool decays, int T, int B, int H, int Hq, int Hk, int Hv, int dk, int dv)
{
    BwdPlan p;
    pad_pair(dk, dv, &p.DK, &p.DV);
    const long long BH = (long long)B * H, rows = (long long)T * BH;
    long long at = 0, most = 0;
    for (int n = 1; n <= 3; ++n) {                         // roles of a launch: fewer are cut into more segments
        int nseg, seg_chunks;
        plan_segments(dtype, T, n * BH, &nseg, &seg_chunks);
        const long long f = passes_floats(n, BH, nseg, p.DK, p.DV);
        most = f > most ? f : most;
    }
    const auto take = [&at](long long n) { const long long o = at; at += up4(n); return o; };
    p.passes = take(most);                                 // of two launches the second begins when the first is done with it
    const long long for_decays = decays ? BH : 0;
    for (long long &keep : p.keep) keep = take(for_decays * anchors(T) * p.DK * p.DV);
    p.flow = take(2 * for_decays * anchors(T));            // doubles
    p.dots = take(2 * for_decays * T);
    p.dq = take(Hq < H ? rows * dk : 0);
    p.dk = take(Hk < H ? rows * dk : 0);
    p.dv = take(Hv < H ? rows * dv : 0);
    p.ds0 = take(for_decays * dk * dv);
    p.end = take(T >= END_FROM ? for_decays * dk * dv : 0);
    p.part = take(2 * for_decays * stretches(T));          // doubles: what they add up to may be far smaller than each
    p.total = at;
    return p;
}

template <typename T>
static void group_sum(const float *in, void *out, int heads, int H, int d, long long total, hipStream_t stream)
{
    const long long blocks = (total + 255) / 256;
    group_sum_kernel<T><<<(unsigned)(blocks < 1 << 20 ? blocks : 1 << 20), 256, 0, stream>>>(in, static_cast<T *>(out), heads, H / heads, d, total);
}

static int group_sum(int dtype, const float *in, void *out, int T, int B, int heads, int H, int d, hipStream_t stream)
{
    const long long total = (long long)T * B * heads * d;
    if (total == 0) return 0;
    if (dtype == DTYPE_BF16) group_sum<__bf16>(in, out, heads, H, d, total, stream);
    else if (dtype == DTYPE_F16) group_sum<_Float16>(in, out, heads, H, d, total, stream);
    else group_sum<float>(in, out, heads, H, d, total, stream);
    return launch_status("linear_attention group sum");
}

template <typename T>
static int launch_step(const void *q, const void *k, const void *v, const float *g, float *state, void *o, const long long *s, int B, int H,
                       int Hq, int Hk, int Hv, int dk, int dv, float scale, hipStream_t stream)
{
    const bool wide = dv % 4 == 0 && (size_t)state % 16 == 0 && s[8] % 4 == 0;
    int zb = dv, nz = 1;                                   // few heads: slices of 16 columns and more
    while ((long long)B * H * nz < 2 * NUM_CU && zb > 16) {
        zb = ((zb + 1) / 2 + 15) & ~15;
        nz = (dv + zb - 1) / zb;
    }
    const int lanes = wide ? (zb + 3) / 4 : zb;
    int lz = 0;
    while ((1 << lz) < lanes) ++lz;
    const dim3 grid((unsigned)(B * H), (unsigned)nz);
    if (wide)
        step_kernel<T, 4><<<grid, 256, 0, stream>>>((const T *)q, (const T *)k, (const T *)v, g, state, (T *)o, s[0], s[1], s[2], s[3], s[4], s[5],
                                                    s[6], s[7], s[8], H, H / Hq, H / Hk, H / Hv, dk, dv, zb, lz, scale);
    else
        step_kernel<T, 1><<<grid, 256, 0, stream>>>((const T *)q, (const T *)k, (const T *)v, g, state, (T *)o, s[0], s[1], s[2], s[3], s[4], s[5],
                                                    s[6], s[7], s[8], H, H / Hq, H / Hk, H / Hv, dk, dv, zb, lz, scale);
    return launch_status("linear_attention_step");
}

}  // namespace la
}  // namespace dmn

using namespace dmn;
using namespace dmn::la;

extern "C" long long dmn_linear_attention_workspace_floats(int dtype, int backward, int T, int B, int H, int Hq, int Hk, int Hv, int dk, int dv)
{
    if (check("dmn_linear_attention_workspace_floats", dtype, T, B, H, Hq, Hk, Hv, dk, dv)) return -1;
    if (backward) return plan_bwd(dtype, backward != 2, T, B, H, Hq, Hk, Hv, dk, dv).total;
    int DC, DZ, nseg, seg_chunks;
    pad_pair(dk, dv, &DC, &DZ);
    plan_segments(dtype, T, (long long)B * H, &nseg, &seg_chunks);
    return passes_floats(1, (long long)B * H, nseg, DC, DZ);
}

extern "C" int dmn_linear_attention_fwd(int dtype, const void *q, const void *k, const void *v, const float *g, const float *state0,
                                        const void *lengths, int lengths64, void *o, float *state, const long long *strides, float *workspace,
                                        int T, int B, int H, int Hq, int Hk, int Hv, int dk, int dv, float scale, void *stream)
{
    const char *who = "dmn_linear_attention_fwd";
    int rc = check(who, dtype, T, B, H, Hq, Hk, Hv, dk, dv);
    if (rc) return rc;
    if (!strides || (B > 0 && T > 0 && (!q || !k || !v || !g || !o))) return fail(-1, "%s: null pointer", who);
    if (!reaches(strides, T, 3)) return fail(-8, "%s: a token's stride must be 0 .. 2^24 + 2^20 elements", who);
    if (B == 0) return 0;
    Args a;
    fill_common(a, g, strides + 9, lengths, lengths64, T, B, H);
    a.nroles = 1;
    int DC, DZ;
    pad_pair(dk, dv, &DC, &DZ);
    plan_segments(dtype, T, (long long)B * H, &a.nseg, &a.seg_chunks);
    if (a.nseg > 1 && (!workspace || (size_t)workspace % 16)) return fail(-7, "%s: this size needs a 16-byte aligned workspace", who);
    Role &r = a.role[0];
    r = Role{};
    r.X = tensor(q, dtype, T, B, Hq, H, dk, strides);
    r.Y = tensor(k, dtype, T, B, Hk, H, dk, strides + 3);
    r.Z = tensor(v, dtype, T, B, Hv, H, dv, strides + 6);
    r.O = dense(o, dtype, T, B, H, dv);
    r.W = r.X;
    r.s_in = state0;
    r.s_out = state;
    r.in_c = r.out_c = dv;
    r.in_z = r.out_z = 1;
    r.dots = nullptr;
    r.scale_p = r.scale_x = scale;
    r.scale_z = 1.0f;
    r.reverse = r.last_decay = 0;
    return run_passes(dtype, a, DC, DZ, 0, workspace, (hipStream_t)stream);
}

extern "C" int dmn_linear_attention_bwd(int dtype, const void *q, const void *k, const void *v, const float *g, const float *state0,
                                        const void *lengths, int lengths64, const void *grad_o, const float *grad_state, void *grad_q, void *grad_k,
                                        void *grad_v, float *grad_g, int grad_g_per_head, float *grad_state0, const long long *strides,
                                        float *workspace, int T, int B, int H, int Hq, int Hk, int Hv, int dk, int dv, float scale, void *stream)
{
    const char *who = "dmn_linear_attention_bwd";
    int rc = check(who, dtype, T, B, H, Hq, Hk, Hv, dk, dv);
    if (rc) return rc;
    if (!strides || (B > 0 && T > 0 && (!q || !k || !v || !g || !grad_o))) return fail(-1, "%s: null pointer", who);
    if (!reaches(strides, T, 3) || !reaches(strides + 12, T, 1)) return fail(-8, "%s: a token's stride must be 0 .. 2^24 + 2^20 elements", who);
    hipStream_t st = (hipStream_t)stream;
    if (B == 0) {
        if (grad_g && grad_g_per_head) {
            decay_grad_heads_kernel<<<(unsigned)H, 64, 0, st>>>(nullptr, grad_g, 0, H, 1);
            return launch_status(who);
        }
        return 0;
    }
    if (!workspace || (size_t)workspace % 16) return fail(-7, "%s: needs a 16-byte aligned workspace", who);
    const BwdPlan p = plan_bwd(dtype, grad_g != nullptr, T, B, H, Hq, Hk, Hv, dk, dv);
    float *dots = workspace + p.dots, *ds0 = grad_state0;
    const bool need_ds0 = grad_state0 || (grad_g && state0);
    if (!ds0) ds0 = workspace + p.ds0;

    const Tensor Q = tensor(q, dtype, T, B, Hq, H, dk, strides), K = tensor(k, dtype, T, B, Hk, H, dk, strides + 3),
                 V = tensor(v, dtype, T, B, Hv, H, dv, strides + 6), D = tensor(grad_o, dtype, T, B, H, H, dv, strides + 12);
    const auto output = [&](void *out, float *ws, int heads, int d) {
        if (!out || heads == H) return dense(out, dtype, T, B, H, d);
        Tensor t = dense(ws, DTYPE_F32, T, B, H, d);
        t.f32 = 1;
        return t;
    };
    const bool meet = grad_g && anchors(T) > 0;           // states of dq and dk between the first and the last
    float *const end = grad_g && grad_state && T >= END_FROM ? workspace + p.end : nullptr;
    Role role[3] = {};
    int n = 0;
    if (grad_q || grad_g) {                               // dq: the operator on (dO, v, k)
        Role &r = role[n++];
        r.X = D; r.Y = V; r.Z = K; r.W = Q;
        r.O = output(grad_q, workspace + p.dq, Hq, dk);
        r.s_in = state0;
        r.s_out = end;
        r.in_c = r.out_c = 1;
        r.in_z = r.out_z = dv;
        r.dots = grad_g ? dots : nullptr;
        r.keep = meet ? workspace + p.keep[0] : nullptr;
        r.scale_p = r.scale_x = scale;
        r.scale_z = 1.0f;
        r.reverse = r.last_decay = 0;
    }
    if (grad_k || grad_g) {                               // dk: backwards in time, on (v, dO, q)
        Role &r = role[n++];
        r.X = V; r.Y = D; r.Z = Q; r.W = K;
        r.O = output(grad_k, workspace + p.dk, Hk, dk);
        r.s_in = grad_state;
        r.s_out = nullptr;
        r.in_c = r.out_c = 1;
        r.in_z = r.out_z = dv;
        r.dots = grad_g ? dots + (size_t)T * B * H : nullptr;
        r.keep = meet ? workspace + p.keep[1] : nullptr;
        r.scale_p = r.scale_z = scale;
        r.scale_x = 1.0f;
        r.reverse = 1;
        r.last_decay = 0;
    }
    const int first = n;
    if (grad_v || need_ds0) {                             // dv and dS_0: backwards in time, on (k, q, dO)
        Role &r = role[n++];
        r.X = K; r.Y = Q; r.Z = D; r.W = V;
        r.O = output(grad_v, workspace + p.dv, Hv, dv);
        r.s_in = grad_state;
        r.s_out = need_ds0 ? ds0 : nullptr;
        r.in_c = r.out_c = dv;
        r.in_z = r.out_z = 1;
        r.dots = nullptr;
        r.scale_p = r.scale_z = scale;
        r.scale_x = 1.0f;
        r.reverse = r.last_decay = 1;
    }
    Args a;
    fill_common(a, g, strides + 9, lengths, lengths64, T, B, H);
    const auto passes = [&](int from, int to, int DC, int DZ, int kind) {
        a.nroles = to - from;
        for (int i = from; i < to; ++i) a.role[i - from] = role[i];
        plan_segments(dtype, T, (long long)a.nroles * B * H, &a.nseg, &a.seg_chunks);
        return from < to ? run_passes(dtype, a, DC, DZ, kind, workspace + p.passes, st) : 0;
    };
    const int dots_too = grad_g ? DOTS_PASS : 0;
    if (p.DK == p.DV) {                                   // all in one launch where keys and values are padded alike
        rc = passes(0, n, p.DV, p.DK, dots_too);
        if (rc) return rc;
    } else {
        rc = passes(0, first, p.DV, p.DK, dots_too);
        if (rc) return rc;
        rc = passes(first, n, p.DK, p.DV, 0);
        if (rc) return rc;
    }
    if (grad_g) {
        double *part = grad_g_per_head ? reinterpret_cast<double *>(workspace + p.part) : nullptr;
        const int ns = stretches(T);
        if (part && T == 0) {
            decay_grad_heads_kernel<<<(unsigned)H, 64, 0, st>>>(nullptr, grad_g, 0, H, 1);
            return launch_status("linear_attention decay gradient");
        }
        double *flow = reinterpret_cast<double *>(workspace + p.flow);
        if (meet) {
            meet_kernel<<<(unsigned)(B * H * anchors(T)), 256, 0, st>>>(reinterpret_cast<const f32x4 *>(workspace + p.keep[0]),
                                                                        reinterpret_cast<const f32x4 *>(workspace + p.keep[1]), flow, p.DK * p.DV / 4);
            rc = launch_status("linear_attention decay gradient");
            if (rc) return rc;
        }
        if (T > 0) {
            decay_scan_kernel<<<(unsigned)(B * H * ns), 256, 0, st>>>(dots, dots + (size_t)T * B * H, flow, state0, ds0, end, grad_state, g, a.gt, a.gb,
                                                                      a.gh, lengths, lengths64, part, T, B, H, dk * dv);
        }
        rc = launch_status("linear_attention decay gradient");
        if (rc) return rc;
        if (!part && T > 0) {
            decay_turn_kernel<<<dim3((unsigned)((T + 63) / 64), (unsigned)((B * H + 63) / 64)), 256, 0, st>>>(dots, g, a.gt, a.gb, a.gh, grad_g, T,
                                                                                                             B * H, H);
            rc = launch_status("linear_attention decay gradient");
            if (rc) return rc;
        }
        if (part) {
            decay_grad_heads_kernel<<<(unsigned)H, 64, 0, st>>>(part, grad_g, B, H, ns);
            rc = launch_status("linear_attention decay gradient");
            if (rc) return rc;
        }
    }
    if (grad_q && Hq < H && (rc = group_sum(dtype, workspace + p.dq, grad_q, T, B, Hq, H, dk, st))) return rc;
    if (grad_k && Hk < H && (rc = group_sum(dtype, workspace + p.dk, grad_k, T, B, Hk, H, dk, st))) return rc;
    if (grad_v && Hv < H && (rc = group_sum(dtype, workspace + p.dv, grad_v, T, B, Hv, H, dv, st))) return rc;
    return 0;
}

extern "C" int dmn_linear_attention_step(int dtype, const void *q, const void *k, const void *v, const float *g, float *state, void *o,
                                         const long long *strides, int B, int H, int Hq, int Hk, int Hv, int dk, int dv, float scale,
                                         void *stream)
{
    const char *who = "dmn_linear_attention_step";
    const int rc = check(who, dtype, 1, B, H, Hq, Hk, Hv, dk, dv);
    if (rc) return rc;
    if (!strides || (B > 0 && (!q || !k || !v || !g || !state || !o))) return fail(-1, "%s: null pointer", who);
    if (B == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DTYPE_BF16) return launch_step<__bf16>(q, k, v, g, state, o, strides, B, H, Hq, Hk, Hv, dk, dv, scale, st);
    if (dtype == DTYPE_F16) return launch_step<_Float16>(q, k, v, g, state, o, strides, B, H, Hq, Hk, Hv, dk, dv, scale, st);
    return launch_step<float>(q, k, v, g, state, o, strides, B, H, Hq, Hk, Hv, dk, dv, scale, st);
}
