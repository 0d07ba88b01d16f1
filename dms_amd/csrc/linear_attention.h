// dms_amd/csrc/linear_attention.h -- what the entry points of linear_attention.hip and the chunk kernels
// (linear_attention.inl, one translation unit for each type) share.
#pragma once
#include "common.h"

namespace dmn {
namespace la {

// One operand: element (t, b, h, c) at p + ((t * st + b * sb + (h / group) * sh + c) * size of an element).
// vec: the widest load that every row allows (2: 16 bytes, 1: 8 bytes, 0: one element).
struct Tensor {
    char *p;
    long long st, sb, sh;
    int d, group, vec, f32;       // f32: fp32 whatever the call's type (outputs that are summed over a group later)
};

// A pass of the recurrence S = a S + y^T z, o = x S over the chunks of a sequence.  The forward operator is one, and
// so is each of its gradients, with other operands in the places of x, y and z and with time running backwards.
struct Role {
    Tensor X, Y, Z, O, W;         // O.p null: not stored.  W.p: dots[t] = sum_c W[t, c] * O[t, c]
    const float *s_in;            // state before the first step, element (c, z) at (b*H + h) * dc*dz + c*in_c + z*in_z, or null
    float *s_out;                 // state after the last step, the same with out_c / out_z, or null
    int in_c, in_z, out_c, out_z;
    float *dots;                  // (B, H, T) or null
    float *keep;                  // with dots: the states that meet another role's at every ANCHOR-th token, or null
    float scale_p, scale_x, scale_z;   // of the products inside a chunk, of x S, and of z in the state
    int reverse;                  // 1: time runs backwards; step s decays by the g of the token after it
    int last_decay;               // 1: s_out is decayed by g of token 0 as well
};

// The gradient of the decays is known from the two states that meet there at every so many tokens, a multiple of both chunks (with
// every 512th, 256 heads of 128 x 128 and 2000 tokens: 2 to 6 % less time, 1.4 times the error).
constexpr int ANCHOR = 256;
__host__ __device__ inline int anchors(int T) { return T > 0 ? (T - 1) / ANCHOR : 0; }

struct Args {
    Role role[3];
    const float *g;
    long long gt, gb, gh;
    const void *lengths;
    int lengths64;
    int T, B, H, nroles, nseg, seg_chunks;
    float *states;                // nseg > 1: (nroles, B*H, nseg) states, each in the kernel's own order
    double *decays;               // nseg > 1: (nroles, B*H, nseg) decay over a segment
};

__device__ __forceinline__ int valid_length(const void *lengths, int lengths64, int b, int T)
{
    if (!lengths) return T;
    const long long n = lengths64 ? static_cast<const long long *>(lengths)[b] : (long long)static_cast<const int *>(lengths)[b];
    return n < 0 ? 0 : (n > T ? T : (int)n);
}

// g in units of log2, with everything that makes 2^g zero in 32 bits (-inf too) at one finite value, so that the
// differences of cumulative sums stay numbers.  NaN stays NaN.
__device__ __forceinline__ double log2_decay(float g)
{
    const double v = (double)g * 1.4426950408889634;
    return v < -160.0 ? -160.0 : v;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double shifted(double v)
{
    const unsigned long long x = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

__device__ __forceinline__ double lane_value(double v, int lane)
{
    const unsigned long long x = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = __builtin_amdgcn_readlane((int)x, lane), hi = __builtin_amdgcn_readlane((int)(x >> 32), lane);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

// inclusive sums over the 64 lanes
__device__ __forceinline__ double lane_sums(double v)
{
    v += shifted<0x111, 0xf>(v);                   // row_shr 1, 2, 4, 8: of 16 lanes
    v += shifted<0x112, 0xf>(v);
    v += shifted<0x114, 0xf>(v);
    v += shifted<0x118, 0xf>(v);
    v += shifted<0x142, 0xa>(v);                   // row_bcast 15, 31: of 64
    v += shifted<0x143, 0xc>(v);
    return v;
}

constexpr int DTYPE_F32 = 0, DTYPE_BF16 = 1, DTYPE_F16 = 2;
inline int elem_size(int dtype) { return dtype == DTYPE_F32 ? 4 : 2; }
// tokens of a chunk: see linear_attention.inl
inline int chunk_tokens(int dtype) { return dtype == DTYPE_BF16 ? 64 : 32; }

// kind, bits:
constexpr int STATES = 1;      // the states after each segment (from s_in for segment 0, from zero for the others), nothing else
constexpr int DOTS_PASS = 2;   // the dots of W and o as well where a role wants them
// DC, DZ (of role[0]) in {32/32, 64/64, 64/128, 128/64, 128/128}.  Returns launch_status.
template <typename T> int launch_chunks(const Args &a, int DC, int DZ, int kind, hipStream_t stream);
extern template int launch_chunks<float>(const Args &, int, int, int, hipStream_t);
extern template int launch_chunks<__bf16>(const Args &, int, int, int, hipStream_t);
extern template int launch_chunks<_Float16>(const Args &, int, int, int, hipStream_t);

}  // namespace la
}  // namespace dmn
