// Appending keys and values to the 8-bit paged cache (fp8_cache.hpp): from
// given rows, or with a layer's q / k RMSNorm and rotation on the way.
//
// Reference behaviour (D3D repository): the KV store of
// serving/vendor/ssd/layers/attention.py:21-22 by slot mapping, q/k
// RMSHeadNorm (layernorm.py:1-52) and rotate-half RoPE
// (rotary_embedding.py:6-16); the reference's cache is bf16.
//
// Per block of tokens that a call touches and KV head, keys and values apart:
//   need = the least e with amax(new finite entries) <= 448 * 2^e
//   the block's first slot is written: e = need, and the slots that the call
//     does not write become 0 (the block starts anew: a page that is used
//     again carries nothing over)
//   else: e = max(old, need), and the kept codes become
//     e4m3(code * 2^(old - e)): exact unless they leave the normal range
//   new code = e4m3(x * 2^-e), |x| past 448 * 2^119 saturated, NaN and
//     infinities as NaN (they do not count in amax)
// A query is normalised and rotated in fp32 and rounded once, to bf16; a key in
// 64 bits and rounded once, to its code.  Angles are position * inv_freq with
// the product and the whole turns taken off in 64 bits.
//
// A (block, head) belongs to one workgroup: of the tokens of a call that fall
// into a block the first in the list leads, its workgroup gathers the others
// wherever they stand (the last of the same slot wins) and does everything
// for the block, so nothing is raced for and results do not depend on order.
// Sixteen lanes hold a row: lane i entries 4i .. 4i + 3 and 64 + 4i .. , the
// pairs that the rotation mixes, or 8i .. 8i + 7 where nothing is rotated.
#include "fp8_cache.hpp"
#include "../../include/d3d_hip.h"

#include <limits.h>

#include <algorithm>
#include <type_traits>

namespace d3d {
namespace fp8 {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_a8 __attribute__((ext_vector_type(4), aligned(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const f32x2_t v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

// Threads that the card holds at once.  While a workgroup per token and KV head
// stays within them, that is the shortest chain; past it a workgroup takes a
// window of tokens and several heads (8 KV heads, appended rows in order: blocks
// of 16 tokens, 128 tokens 4.9 us against 5.9, 256 5.4 against 6.0, 400 7.3
// against 6.1; blocks of 64, 64 tokens 6.8 against 8.5, 256 12.4 against 8.0).
constexpr int64_t kCardThreads = 256 * 2048;
constexpr int kManyHeads = 8;   // query heads of a token that 8 lanes take, where tokens are many
constexpr float kMaxValue = 448.f * 0x1p119f;  // 448 * 2^kMaxExp

struct AppendParams {
    // Rows: k and v [T] of Hkv heads (token strides in entries); the rotating
    // form's are parts of qkv [T, Hq + 2 Hkv] heads, bf16 or fp32 partials.
    const uint16_t* qkv;
    const uint16_t* k;
    const uint16_t* v;
    int64_t k_stride, v_stride;
    const float* parts;
    int splits;
    size_t part_stride;
    const int64_t* positions;
    const uint16_t* qn;
    const uint16_t* kn;
    const float* inv_freq;
    uint16_t* q_out;
    float eps;
    uint8_t* k_cache;
    uint8_t* v_cache;
    uint8_t* k_scale;
    uint8_t* v_scale;
    const int64_t* slots;
    int T, Hq, Hkv, page_size, block_shift;
    int64_t num_slots;
    int win;       // tokens per key / value workgroup, at most 64
    int kv_heads;  // KV heads per key / value workgroup
    int kv_groups; // workgroups of keys and values; queries follow
};

// Entries 4i .. 4i + 3 of a bf16 row.
__device__ __forceinline__ void unpack4(u32x2 r, float* x) {
    x[0] = __uint_as_float(r[0] << 16);
    x[1] = __uint_as_float(r[0] & 0xffff0000u);
    x[2] = __uint_as_float(r[1] << 16);
    x[3] = __uint_as_float(r[1] & 0xffff0000u);
}

// A row's entries of lane i of 16 as bf16.  Rotating: r[0] = 4i .. 4i + 3, r[1] =
// 64 + 4i .. , a pair's two in one lane; else 8i .. 8i + 7, one piece of memory.
template <bool ROPE, bool PARTS>
__device__ __forceinline__ void load_row(const uint16_t* src, const AppendParams& P, size_t e, int i, u32x2* r) {
    if constexpr (!ROPE) {
        const u32x4_a8 v = *reinterpret_cast<const u32x4_a8*>(src + 8 * i);
        r[0] = u32x2{v[0], v[1]};
        r[1] = u32x2{v[2], v[3]};
    } else if constexpr (PARTS) {
        f32x4 a = *reinterpret_cast<const f32x4*>(P.parts + e + 4 * i);
        f32x4 b = *reinterpret_cast<const f32x4*>(P.parts + e + 64 + 4 * i);
        for (int sp = 1; sp < P.splits; ++sp) {
            const float* q = P.parts + (size_t)sp * P.part_stride + e;
            a += *reinterpret_cast<const f32x4*>(q + 4 * i);
            b += *reinterpret_cast<const f32x4*>(q + 64 + 4 * i);
        }
        // The product's value is the partials' sum rounded to bf16.
        r[0] = u32x2{pack2(a[0], a[1]), pack2(a[2], a[3])};
        r[1] = u32x2{pack2(b[0], b[1]), pack2(b[2], b[3])};
    } else {
        r[0] = *reinterpret_cast<const u32x2*>(src + 4 * i);
        r[1] = *reinterpret_cast<const u32x2*>(src + 64 + 4 * i);
    }
}

// cos and sin of position * f, where p = position / 2 pi: the angle in turns in
// 64 bits, whole turns and then quarters taken off, and Taylor sums of the rest
// x, |x| <= pi / 4, whose next terms x^11 / 11! and x^12 / 12! are below 2^-29 and
// 2^-33; what a float leaves of x goes in by the derivative.
__device__ __forceinline__ void cos_sin(double p, float f, float& cs, float& sn) {
    double turns = p * (double)f;
    turns = 4.0 * (turns - rint(turns));
    const double q = rint(turns), xd = (turns - q) * 1.57079632679489661923;
    const float x = (float)xd, dx = (float)(xd - (double)x), z = x * x;
    const float s0 = x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
    const float c0 = z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 - z * (1.f / 3628800)))));
    const float s = x + (s0 + dx), c = 1.f + (c0 - x * dx);
    const int k = (int)q;  // -2 .. 2 quarters
    cs = (k & 1) ? s : c;
    sn = (k & 1) ? c : s;
    if ((k + 1) & 2) cs = -cs;
    if (k & 2) sn = -sn;
}

// The same in 64 bits, with the sums' next terms below 2^-45 and 2^-49.
__device__ __forceinline__ void cos_sin(double p, float f, double& cs, double& sn) {
    double turns = p * (double)f;
    turns = 4.0 * (turns - rint(turns));
    const double q = rint(turns), x = (turns - q) * 1.57079632679489661923, z = x * x;
    double s = 1.0 / 6227020800, c = -1.0 / 87178291200;
    s = __builtin_fma(s, z, -1.0 / 39916800);
    c = __builtin_fma(c, z, 1.0 / 479001600);
    s = __builtin_fma(s, z, 1.0 / 362880);
    c = __builtin_fma(c, z, -1.0 / 3628800);
    s = __builtin_fma(s, z, -1.0 / 5040);
    c = __builtin_fma(c, z, 1.0 / 40320);
    s = __builtin_fma(s, z, 1.0 / 120);
    c = __builtin_fma(c, z, -1.0 / 720);
    s = __builtin_fma(s, z, -1.0 / 6);
    c = __builtin_fma(c, z, 1.0 / 24);
    s = __builtin_fma(x * z, s, x);
    c = __builtin_fma(c, z, -0.5);
    c = __builtin_fma(c, z, 1.0);
    const int k = (int)q;
    cs = (k & 1) ? s : c;
    sn = (k & 1) ? c : s;
    if ((k + 1) & 2) cs = -cs;
    if (k & 2) sn = -sn;
}

constexpr double kTurn = 0.15915494309189533577;  // 1 / 2 pi

template <int N, typename T>
__device__ __forceinline__ void angles(const AppendParams& P, int64_t pos, int e, T* cs, T* sn) {
    const double p = (double)pos * kTurn;
#pragma unroll
    for (int j = 0; j < N; ++j) cos_sin(p, P.inv_freq[e + j], cs[j], sn[j]);
}

// A query row's RMSNorm over its 8 lanes (each with 8 entries and their
// partners 64 further), then the rotation.
__device__ __forceinline__ void norm_rotate_q(float* x, const float* w, const float* cs, const float* sn, float eps) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) ss = __builtin_fmaf(x[j], x[j], ss);
    ss += xor_asc<1>(ss);
    ss += xor_asc<2>(ss);
    ss += xor_asc<4>(ss);
    const float rstd = rsqrtf(ss / (float)D + eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float a = x[j] * rstd * w[j], b = x[8 + j] * rstd * w[8 + j];
        x[j] = a * cs[j] - b * sn[j];
        x[8 + j] = b * cs[j] + a * sn[j];
    }
}

template <int O>
__device__ __forceinline__ double xor_desc_d(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = xor_partner_desc<O>((uint32_t)u), hi = xor_partner_desc<O>((uint32_t)(u >> 32));
    return __builtin_bit_cast(double, hi << 32 | lo);
}

// x as a float rounded to odd: cut off, with the last bit set if anything was.  A
// rounding of it to fewer bits, and a comparison, then comes out as x's own would.
__device__ __forceinline__ float to_odd(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)u, kept = lo & 0xe0000000u;
    const uint64_t v = (u >> 32 << 32) | ((lo & 0x1fffffffu) ? kept | 0x20000000u : kept);
    return (float)__builtin_bit_cast(double, v);
}

// A key row's, over 16 lanes with 4 entries and their partners.  A key is
// rounded to 4 bits, so a value next to a border falls to another code by any
// error: the sum, the root (one Newton step on the hardware's) and the
// rotation of x w, which a float holds exactly, run in 64 bits.
__device__ __forceinline__ void norm_rotate_k(float* x, const float* w, const double* cs, const double* sn, float eps) {
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)x[j], (double)x[j], ss);
    ss += xor_desc_d<8>(ss);
    ss += xor_desc_d<4>(ss);
    ss += xor_desc_d<2>(ss);
    ss += xor_desc_d<1>(ss);
    const double v = ss * (1.0 / D) + (double)eps;
    const double r0 = (double)rsqrtf((float)v);
    const double r = __builtin_fma(0.5 * r0, __builtin_fma(-v * r0, r0, 1.0), r0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double a = (double)(x[j] * w[j]), b = (double)(x[4 + j] * w[4 + j]);
        x[j] = to_odd((a * cs[j] - b * sn[j]) * r);
        x[4 + j] = to_odd((b * cs[j] + a * sn[j]) * r);
    }
}

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;
}

// The largest |x| of entries that are finite, NaN or (then the result is not
// finite) infinite; of bf16 pairs, as integers.
__device__ __forceinline__ float amax_f32(const float* x) {
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) a = fmaxf(a, fabsf(x[j]));
    return a;
}
__device__ __forceinline__ float amax_bf16(const u32x2* r) {
    u16x2 a = __builtin_bit_cast(u16x2, r[0][0] & 0x7fff7fffu);
    a = __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, r[0][1] & 0x7fff7fffu));
    a = __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, r[1][0] & 0x7fff7fffu));
    a = __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, r[1][1] & 0x7fff7fffu));
    return __uint_as_float((uint32_t)max(a[0], a[1]) << 16);
}

// x * 2^-e as codes: to nearest even, NaN and infinities to NaN.  Only the
// largest exponent can leave a finite entry past 448: it is clamped there.
__device__ __forceinline__ uint32_t quantise(const float* x, int e) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        y[j] = x[j];
        if (e == kMaxExp && fabsf(x[j]) < INFINITY) y[j] = fminf(fmaxf(y[j], -kMaxValue), kMaxValue);
    }
    s16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, y[0], y[1], pow2(e), false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, y[2], y[3], pow2(e), true);
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ uint32_t quantise(u32x2 x, int e) {
    if (e == kMaxExp) {  // uniform
        float y[4];
        unpack4(x, y);
        return quantise(y, e);
    }
    const uint32_t lo = x[0], hi = x[1];  // a bit cast of a vector's element takes element 0
    s16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, lo), pow2(e), false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, hi), pow2(e), true);
    return __builtin_bit_cast(uint32_t, r);
}

// Eight kept codes of a row under a scale 2^d times finer (f = 2^d, d <= 0).
__device__ __forceinline__ uint32_t rescale(uint32_t c, float f) {
    const float y0 = __builtin_amdgcn_cvt_f32_fp8((int)c, 0), y1 = __builtin_amdgcn_cvt_f32_fp8((int)c, 1);
    const float y2 = __builtin_amdgcn_cvt_f32_fp8((int)c, 2), y3 = __builtin_amdgcn_cvt_f32_fp8((int)c, 3);
    return codes4(y0 * f, y1 * f, y2 * f, y3 * f);
}
__device__ __forceinline__ void rescale_row(uint8_t* row, int i, float f) {
    u32x2* at = reinterpret_cast<u32x2*>(row) + i;
    const u32x2 c = *at;
    *at = u32x2{rescale(c[0], f), rescale(c[1], f)};
}

// Lane i's codes of a row: of the entries that load_row gave it.
template <bool ROPE>
__device__ __forceinline__ void put_codes(uint8_t* row, int i, uint32_t a, uint32_t b) {
    if constexpr (ROPE) {
        reinterpret_cast<uint32_t*>(row)[i] = a;
        reinterpret_cast<uint32_t*>(row)[16 + i] = b;
    } else {
        reinterpret_cast<u32x2*>(row)[i] = u32x2{a, b};
    }
}

// A query row's entries of lane i of 8: x[0..7] = 8i .., x[8..15] = 64 + 8i ...
template <bool PARTS>
__device__ __forceinline__ void load_row8(const uint16_t* src, const AppendParams& P, size_t e, int i, float* x) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
        if constexpr (PARTS) {
            const float* q = P.parts + e + 64 * hf + 8 * i;
            f32x4 a = *reinterpret_cast<const f32x4*>(q), b = *reinterpret_cast<const f32x4*>(q + 4);
            for (int sp = 1; sp < P.splits; ++sp) {
                q += P.part_stride;
                a += *reinterpret_cast<const f32x4*>(q);
                b += *reinterpret_cast<const f32x4*>(q + 4);
            }
            unpack4(u32x2{pack2(a[0], a[1]), pack2(a[2], a[3])}, x + 8 * hf);
            unpack4(u32x2{pack2(b[0], b[1]), pack2(b[2], b[3])}, x + 8 * hf + 4);
        } else {
            const u32x4_a8 r = *reinterpret_cast<const u32x4_a8*>(src + 64 * hf + 8 * i);
            unpack4(u32x2{r[0], r[1]}, x + 8 * hf);
            unpack4(u32x2{r[2], r[3]}, x + 8 * hf + 4);
        }
    }
}

// HP heads at a time, each by NT / HP threads that take NT / HP / 16 slots of a
// block at a time, IT times.  MANY: two workgroups of 512 threads per CU, within
// 128 registers (7,800 tokens of 32 + 8 heads 38 us, with 130 registers 48).
//
// What bounds it: many tokens, their bytes (that call's 176 MB at 4.6 TB/s; 14,688
// tokens of 8 heads, 90 MB, 31 us at 2.9 TB/s: 459 windows are fewer than two per
// CU, and more workgroups would each read the call's slots again).  Few, the chain
// slots, block, rows, largest, codes (16 tokens of 32 + 8 heads 5.1 us).
template <bool MANY, int NT, int HP, int IT, bool ROPE, bool PARTS>
__global__ __launch_bounds__(NT, MANY ? 4 : 1) void append_kernel(AppendParams P) {
    const int tid = threadIdx.x, i16 = tid & 15;
    if constexpr (ROPE) {
        if ((int)blockIdx.x >= P.kv_groups) {
            // Queries: 8 lanes take QH heads of one token, QB rows on the way together (two
            // 38.2 us for 7,800 tokens, one 39.2; four 38.5, eight run out of registers).
            constexpr int QH = MANY ? kManyHeads : 1, QB = MANY ? 2 : 1;
            const int i8 = tid & 7;
            const int chunks = (P.Hq + QH - 1) / QH;
            const int64_t g = (int64_t)((int)blockIdx.x - P.kv_groups) * (NT / 8) + (tid >> 3);
            const bool live = g < (int64_t)P.T * chunks;
            const int t = live ? (int)(g / chunks) : 0, h0 = live ? (int)(g % chunks) * QH : 0;
            float cs[8], sn[8], w[16];
            angles<8>(P, P.positions[t], 8 * i8, cs, sn);
            load_row8<false>(P.qn, P, 0, i8, w);
            const int n = min(QH, P.Hq - h0);
#pragma unroll
            for (int jb = 0; jb < QH; jb += QB) {
                float x[QB][16];
#pragma unroll
                for (int c = 0; c < QB; ++c) {  // behind the last head: the last one again, not written
                    const size_t e = ((size_t)t * (P.Hq + 2 * P.Hkv) + h0 + min(jb + c, n - 1)) * D;
                    load_row8<PARTS>(P.qkv + e, P, e, i8, x[c]);
                }
#pragma unroll
                for (int c = 0; c < QB; ++c) {
                    norm_rotate_q(x[c], w, cs, sn, P.eps);
                    if (live && jb + c < n) {
                        uint16_t* dst = P.q_out + ((size_t)t * P.Hq + h0 + jb + c) * D + 8 * i8;
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            const float* y = x[c] + 8 * hf;
                            *reinterpret_cast<u32x4_a8*>(dst + 64 * hf) =
                                u32x4_a8{pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7])};
                        }
                    }
                }
            }
            return;
        }
    }
    __shared__ int member[kMaxBlock];  // per slot of the block: the token that writes it, or -1
    __shared__ float red[2][2][NT / kWave];
    const int h_groups = (P.Hkv + P.kv_heads - 1) / P.kv_heads;
    const int h_first = (int)(blockIdx.x % h_groups) * P.kv_heads, h_last = min(h_first + P.kv_heads, P.Hkv);
    const int t_first = (int)(blockIdx.x / h_groups) * P.win;
    const int block = 1 << P.block_shift, per_page = P.page_size >> P.block_shift;
    constexpr int ROWS = NT / HP / 16, HW = NT / HP / kWave;  // slots and waves of a head at a time
    const int lane = tid & 63, row16 = (tid >> 4) % ROWS, hp = tid / (NT / HP);
    // The window's tokens that follow one of another block lead a run; every
    // wave finds them (win <= 64).
    const auto block_of = [&](int64_t s) { return s >= 0 && s < P.num_slots ? s >> P.block_shift : (int64_t)-1; };
    int64_t mine = -1, prev = -1;
    if (lane < P.win && t_first + lane < P.T) {
        mine = block_of(P.slots[t_first + lane]);
        if (t_first + lane > 0) prev = block_of(P.slots[t_first + lane - 1]);
    }
    uint64_t lead = __ballot(mine >= 0 && mine != prev);
    for (; lead; lead &= lead - 1) {  // uniform over the workgroup
        const int src = __builtin_ctzll(lead), t = t_first + src;
        const int64_t blk = (int64_t)__shfl((unsigned long long)mine, src, 64);
        for (int j = tid; j < block; j += NT) member[j] = -1;
        __syncthreads();
        // One pass over the call's slots: its tokens of this block, wherever they stand.
        // Up to sixteen loads at a time are on the way together (14,688 tokens: 42 -> 29
        // us), and their slots are looked at one by one only where one of them is the
        // block's (128 tokens of 8 heads 6.3 -> 5.4 us, 512 8.0 -> 6.1).
        bool before = false;
        const uint64_t at = (uint64_t)blk << P.block_shift;
        const uint32_t at_lo = (uint32_t)at, at_hi = (uint32_t)(at >> 32), keep = ~(uint32_t)(block - 1);
        const auto scan = [&](int j0, auto n, auto full) {
            constexpr int N = decltype(n)::value;
            uint32_t lo[N], hi[N], best = ~0u;
#pragma unroll
            for (int i = 0; i < N; ++i) {  // behind the last token: the last one again, which changes nothing
                const int j = j0 + i * NT + tid;
                const uint64_t s = (uint64_t)P.slots[decltype(full)::value ? j : min(j, P.T - 1)];
                lo[i] = (uint32_t)s;
                hi[i] = (uint32_t)(s >> 32);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) best = min(best, ((lo[i] ^ at_lo) & keep) | (hi[i] ^ at_hi));
            if (best == 0) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int j = min(j0 + i * NT + tid, P.T - 1);
                    if ((((lo[i] ^ at_lo) & keep) | (hi[i] ^ at_hi)) == 0) {
                        before |= j < t;
                        atomicMax(&member[lo[i] & (block - 1)], j);
                    }
                }
            }
        };
        int j0 = 0;
        for (; P.T - j0 >= 16 * NT; j0 += 16 * NT) scan(j0, std::integral_constant<int, 16>{}, std::true_type{});
        if (P.T - j0 > 4 * NT)
            scan(j0, std::integral_constant<int, 16>{}, std::false_type{});
        else if (P.T - j0 > NT)
            scan(j0, std::integral_constant<int, 4>{}, std::false_type{});
        else if (P.T > j0)
            scan(j0, std::integral_constant<int, 1>{}, std::false_type{});
        if (__syncthreads_or(before)) continue;  // an earlier token leads this block
        const int64_t page = blk / per_page;
        const int nb = (int)(blk - page * per_page);
        const bool anew = member[0] >= 0;
        int m[IT];
        bool some[IT];  // of the wave's rows one is written; of many tokens they mostly are, and asking costs registers
        // With one row per thread its angles stay, and the next heads' rows are on the
        // way while these are worked on; with more the registers do not reach.
        constexpr bool KEEP = IT == 1, AHEAD = KEEP && MANY;
        double cs[4], sn[4];
        float w[8];
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            m[it] = member[row16 + it * ROWS];
            some[it] = MANY || __any(m[it] >= 0);
        }
        if constexpr (ROPE) {
            u32x2 r[2];
            load_row<true, false>(P.kn, P, 0, i16, r);
            unpack4(r[0], w);
            unpack4(r[1], w + 4);
            if (KEEP && some[0]) angles<4>(P, P.positions[max(m[0], 0)], 4 * i16, cs, sn);
        }
        u32x2 raw[IT][4];
        int old_k = 0, old_v = 0;
        const auto head_at = [&](int hb) { return min(hb + hp, h_last - 1); };
        const auto fetch = [&](int h) {
            const size_t sc = ((size_t)page * P.Hkv + h) * per_page + nb;
            old_k = P.k_scale[sc];
            old_v = P.v_scale[sc];
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                if (!some[it]) continue;
                const size_t tm = (size_t)max(m[it], 0), e = (tm * (P.Hq + 2 * P.Hkv) + P.Hq + h) * D;
                load_row<ROPE, PARTS>(P.k + tm * P.k_stride + (size_t)h * D, P, e, i16, raw[it]);
                load_row<ROPE, PARTS>(P.v + tm * P.v_stride + (size_t)h * D, P, e + (size_t)P.Hkv * D, i16, raw[it] + 2);
            }
        };
        if constexpr (AHEAD) fetch(head_at(h_first));
        for (int hb = h_first; hb < h_last; hb += HP) {
            const bool here = hb + hp < h_last;
            const int h = head_at(hb);
            const size_t row0 = ((size_t)page * P.Hkv + h) * P.page_size + (size_t)nb * block;
            const size_t sc = ((size_t)page * P.Hkv + h) * per_page + nb;
            if constexpr (!AHEAD) fetch(h);
            float xk[ROPE ? IT : 1][8];
            u32x2 rk[IT][2], rv[IT][2];
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                rk[it][0] = raw[it][0];
                rk[it][1] = raw[it][1];
                rv[it][0] = raw[it][2];
                rv[it][1] = raw[it][3];
            }
            const int was_k = min(old_k - 127, kMaxExp), was_v = min(old_v - 127, kMaxExp);
            if constexpr (AHEAD) {
                if (hb + HP < h_last) fetch(head_at(hb + HP));
            }
            float ak = 0.f, av = 0.f;
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                if (!some[it]) continue;
                float a, v = amax_bf16(rv[it]);
                if constexpr (ROPE) {
                    unpack4(rk[it][0], xk[it]);
                    unpack4(rk[it][1], xk[it] + 4);
                    if constexpr (!KEEP) angles<4>(P, P.positions[max(m[it], 0)], 4 * i16, cs, sn);
                    norm_rotate_k(xk[it], w, cs, sn, P.eps);
                    a = amax_f32(xk[it]);
                } else {
                    a = amax_bf16(rk[it]);
                }
                if (__any(!(a < INFINITY) || !(v < INFINITY))) {  // something is not finite: it does not count
                    float x[8];
                    unpack4(rv[it][0], x);
                    unpack4(rv[it][1], x + 4);
                    v = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) v = fmaxf(v, finite_abs(x[j]));
                    unpack4(rk[it][0], x);
                    unpack4(rk[it][1], x + 4);
                    a = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) a = fmaxf(a, finite_abs(ROPE ? xk[it][j] : x[j]));
                }
                ak = fmaxf(ak, m[it] >= 0 ? a : 0.f);
                av = fmaxf(av, m[it] >= 0 ? v : 0.f);
            }
            ak = wave_max(ak);
            av = wave_max(av);
            const int odd = ((hb - h_first) / HP) & 1;  // two sets: the next heads' maxima do not wait for these ones' readers
            if (lane == 0) {
                red[odd][0][tid >> 6] = ak;
                red[odd][1][tid >> 6] = av;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < HW; ++i) {
                ak = fmaxf(ak, red[odd][0][hp * HW + i]);
                av = fmaxf(av, red[odd][1][hp * HW + i]);
            }
            // Uniform over the head's waves.
            const int ek = __builtin_amdgcn_readfirstlane(anew ? need_exp(ak) : max(was_k, need_exp(ak)));
            const int ev = __builtin_amdgcn_readfirstlane(anew ? need_exp(av) : max(was_v, need_exp(av)));
            // Kept codes shrink by 2^(was - new): past 2^-20 nothing is left of 448.
            const float fk = pow2(max(was_k - ek, -20)), fv = pow2(max(was_v - ev, -20));
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                const int r = row16 + it * ROWS;
                uint8_t* dk = P.k_cache + (row0 + r) * D;
                uint8_t* dv = P.v_cache + (row0 + r) * D;
                if (!here) continue;
                if (m[it] >= 0) {
                    if constexpr (ROPE)
                        put_codes<ROPE>(dk, i16, quantise(xk[it], ek), quantise(xk[it] + 4, ek));
                    else
                        put_codes<ROPE>(dk, i16, quantise(rk[it][0], ek), quantise(rk[it][1], ek));
                    put_codes<ROPE>(dv, i16, quantise(rv[it][0], ev), quantise(rv[it][1], ev));
                } else if (anew) {
                    put_codes<ROPE>(dk, i16, 0u, 0u);
                    put_codes<ROPE>(dv, i16, 0u, 0u);
                } else {
                    if (ek != was_k) rescale_row(dk, i16, fk);
                    if (ev != was_v) rescale_row(dv, i16, fv);
                }
            }
            // Every thread has read the old scales before this head's barrier.
            if (here && tid % (NT / HP) == 0) {
                P.k_scale[sc] = (uint8_t)(ek + 127);
                P.v_scale[sc] = (uint8_t)(ev + 127);
            }
        }
        __syncthreads();  // member is used again
    }
}

template <bool MANY, int NT, int HP, int IT, bool ROPE, bool PARTS>
static int launch(AppendParams& P, hipStream_t s) {
    // Few tokens: a workgroup per token and head, for the shortest chain.  Many:
    // windows of a block's tokens and all of a workgroup's heads in one pass over the
    // call's slots, split further while there are fewer workgroups than CUs.
    P.win = MANY ? std::min(1 << P.block_shift, 64) : 1;
    const int64_t windows = ((int64_t)P.T + P.win - 1) / P.win;
    const int rounds = (P.Hkv + HP - 1) / HP;
    P.kv_heads = MANY ? HP * (int)std::min<int64_t>(rounds, std::max<int64_t>(1, windows * rounds / 256)) : 1;
    int64_t groups = windows * ((P.Hkv + P.kv_heads - 1) / P.kv_heads);
    if (groups > INT_MAX) return D3D_E_SHAPE;
    P.kv_groups = (int)groups;
    if (ROPE) {
        constexpr int QH = MANY ? kManyHeads : 1;
        const int64_t chunks = (P.Hq + QH - 1) / QH;
        groups += ((int64_t)P.T * chunks + NT / 8 - 1) / (NT / 8);
    }
    if (groups > (int64_t)UINT32_MAX / NT) return D3D_E_SHAPE;  // threads of a launch
    hipLaunchKernelGGL((append_kernel<MANY, NT, HP, IT, ROPE, PARTS>), dim3((unsigned)groups), dim3(NT), 0, s, P);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? D3D_OK : (int)err;
}

template <bool ROPE, bool PARTS>
static int run(AppendParams& P, void* stream) {
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int threads = std::min(16 << P.block_shift, 1024);  // of a workgroup for one token and head
    const bool many = (int64_t)P.T * P.Hkv * threads > kCardThreads;
    switch (P.block_shift) {
        case 4:
            return many ? launch<true, 512, 2, 1, ROPE, PARTS>(P, s) : launch<false, 256, 1, 1, ROPE, PARTS>(P, s);
        case 5: return many ? launch<true, 512, 1, 1, ROPE, PARTS>(P, s) : launch<false, 512, 1, 1, ROPE, PARTS>(P, s);
        case 6:
            return many ? launch<true, 1024, 1, 1, ROPE, PARTS>(P, s) : launch<false, 1024, 1, 1, ROPE, PARTS>(P, s);
        case 7:
            return many ? launch<true, 1024, 1, 2, ROPE, PARTS>(P, s) : launch<false, 1024, 1, 2, ROPE, PARTS>(P, s);
        default:
            return many ? launch<true, 1024, 1, 4, ROPE, PARTS>(P, s) : launch<false, 1024, 1, 4, ROPE, PARTS>(P, s);
    }
}

static bool off(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

// The cache's part of the arguments.
static int cache_args(AppendParams& P, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                      const int64_t* slots, int T, int Hkv, int D_, int page_size, int block, int num_pages) {
    if (T < 0 || T > 1 << 30 || Hkv < 1 || page_size < 1 || num_pages < 1) return D3D_E_SHAPE;
    if (D_ != D) return D3D_E_UNSUPPORTED;
    const int sh = fp8_block_shift(page_size, block);
    if (sh < 0) return D3D_E_UNSUPPORTED;
    if (T == 0) return D3D_OK;
    if (!k_cache || !v_cache || !k_scale || !v_scale || !slots) return D3D_E_NULL;
    if (off(k_cache, 16) || off(v_cache, 16)) return D3D_E_UNSUPPORTED;
    P.k_cache = static_cast<uint8_t*>(k_cache);
    P.v_cache = static_cast<uint8_t*>(v_cache);
    P.k_scale = static_cast<uint8_t*>(k_scale);
    P.v_scale = static_cast<uint8_t*>(v_scale);
    P.slots = slots;
    P.T = T;
    P.Hkv = Hkv;
    P.page_size = page_size;
    P.block_shift = sh;
    P.num_slots = (int64_t)num_pages * page_size;
    return D3D_OK;
}

static int rope(const void* qkv, const float* parts, int splits, const int64_t* positions, const void* q_norm_w,
                const void* k_norm_w, const float* inv_freq, void* q_out, void* k_cache, void* v_cache, void* k_scale,
                void* v_scale, const int64_t* slots, int T, int Hq, int Hkv, int D_, float eps, int page_size,
                int block, int num_pages, void* stream) {
    AppendParams P{};
    if (Hq < 1) return D3D_E_SHAPE;
    const int st = cache_args(P, k_cache, v_cache, k_scale, v_scale, slots, T, Hkv, D_, page_size, block, num_pages);
    if (st != D3D_OK || T == 0) return st;
    if ((!qkv && !parts) || !positions || !q_norm_w || !k_norm_w || !inv_freq || !q_out) return D3D_E_NULL;
    if (off(qkv, 8) || off(parts, 16) || off(q_norm_w, 8) || off(k_norm_w, 8) || off(inv_freq, 16) || off(q_out, 8))
        return D3D_E_UNSUPPORTED;
    P.qkv = static_cast<const uint16_t*>(qkv);
    if (qkv) {
        P.k = P.qkv + (size_t)Hq * D;
        P.v = P.k + (size_t)Hkv * D;
    }
    P.k_stride = P.v_stride = (int64_t)(Hq + 2 * Hkv) * D;
    P.parts = parts;
    P.splits = splits;
    P.part_stride = (size_t)T * (Hq + 2 * Hkv) * D;
    P.positions = positions;
    P.qn = static_cast<const uint16_t*>(q_norm_w);
    P.kn = static_cast<const uint16_t*>(k_norm_w);
    P.inv_freq = inv_freq;
    P.q_out = static_cast<uint16_t*>(q_out);
    P.eps = eps;
    P.Hq = Hq;
    return parts ? run<true, true>(P, stream) : run<true, false>(P, stream);
}

}  // namespace fp8
}  // namespace d3d

using namespace d3d;

extern "C" int d3d_kv_append_fp8(const void* k, const void* v, int64_t k_stride, int64_t v_stride, void* k_cache,
                                 void* v_cache, void* k_scale, void* v_scale, const int64_t* slot_mapping,
                                 int n_tokens, int Hkv, int D, int page_size, int block, int num_pages,
                                 void* stream) {
    fp8::AppendParams P{};
    const int st = fp8::cache_args(P, k_cache, v_cache, k_scale, v_scale, slot_mapping, n_tokens, Hkv, D, page_size,
                                   block, num_pages);
    if (st != D3D_OK || n_tokens == 0) return st;
    if (!k || !v) return D3D_E_NULL;
    if (k_stride < 0 || v_stride < 0 || k_stride % 4 || v_stride % 4 || fp8::off(k, 8) || fp8::off(v, 8))
        return D3D_E_UNSUPPORTED;
    P.k = static_cast<const uint16_t*>(k);
    P.v = static_cast<const uint16_t*>(v);
    P.k_stride = k_stride;
    P.v_stride = v_stride;
    return fp8::run<false, false>(P, stream);
}

extern "C" int d3d_qk_rope_append_fp8(const void* qkv, const int64_t* positions, const void* q_norm_w,
                                      const void* k_norm_w, const float* inv_freq, void* q_out, void* k_cache,
                                      void* v_cache, void* k_scale, void* v_scale, const int64_t* slot_mapping, int T,
                                      int Hq, int Hkv, int D, float eps, int page_size, int block, int num_pages,
                                      void* stream) {
    return fp8::rope(qkv, nullptr, 0, positions, q_norm_w, k_norm_w, inv_freq, q_out, k_cache, v_cache, k_scale,
                     v_scale, slot_mapping, T, Hq, Hkv, D, eps, page_size, block, num_pages, stream);
}

extern "C" int d3d_qk_rope_append_fp8_parts(const float* parts, int splits, const int64_t* positions,
                                            const void* q_norm_w, const void* k_norm_w, const float* inv_freq,
                                            void* q_out, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                                            const int64_t* slot_mapping, int T, int Hq, int Hkv, int D, float eps,
                                            int page_size, int block, int num_pages, void* stream) {
    if (splits < 1) return D3D_E_SHAPE;
    return fp8::rope(nullptr, parts, splits, positions, q_norm_w, k_norm_w, inv_freq, q_out, k_cache, v_cache, k_scale,
                     v_scale, slot_mapping, T, Hq, Hkv, D, eps, page_size, block, num_pages, stream);
}
