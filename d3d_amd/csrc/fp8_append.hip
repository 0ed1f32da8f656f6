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
// Norm, rotation and scaling run in fp32 and a key is rounded once, to its
// code; a query once, to bf16.  Angles are position * inv_freq with the
// product and the whole turns taken off in 64 bits.
//
// A workgroup owns one (block, head): of the tokens of a call that fall into a
// block the first in the list leads, its workgroup gathers the others
// wherever they stand (the last of the same slot wins) and does everything
// for the block, so nothing is raced for and results do not depend on order.
// Sixteen lanes hold a row: lane i entries 4i .. 4i + 3 and 64 + 4i .. , the
// pairs that the rotation mixes.
#include "fp8_cache.hpp"
#include "../../include/d3d_hip.h"

#include <limits.h>

namespace d3d {
namespace fp8 {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const f32x2_t v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

struct AppendParams {
    // Rows: k and v [T] of Hkv heads (token strides in entries), or for the
    // rotating form qkv [T, Hq + 2 Hkv] heads, as bf16 or as fp32 partials.
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
    int win;       // tokens per key / value workgroup
    int kv_groups; // workgroups of keys and values; queries follow
    int q_heads;   // query heads per 16 lanes
};

// Entries 4i .. 4i + 3 of a bf16 row.
__device__ __forceinline__ void unpack4(u32x2 r, float* x) {
    x[0] = __uint_as_float(r[0] << 16);
    x[1] = __uint_as_float(r[0] & 0xffff0000u);
    x[2] = __uint_as_float(r[1] << 16);
    x[3] = __uint_as_float(r[1] & 0xffff0000u);
}

// A row's entries of lane i: x[0..3] = 4i .., x[4..7] = 64 + 4i ...
template <bool PARTS>
__device__ __forceinline__ void load_row(const uint16_t* src, const AppendParams& P, size_t e, int i, float* x) {
    if constexpr (PARTS) {
        f32x4 a = *reinterpret_cast<const f32x4*>(P.parts + e + 4 * i);
        f32x4 b = *reinterpret_cast<const f32x4*>(P.parts + e + 64 + 4 * i);
        for (int sp = 1; sp < P.splits; ++sp) {
            const float* q = P.parts + (size_t)sp * P.part_stride + e;
            a += *reinterpret_cast<const f32x4*>(q + 4 * i);
            b += *reinterpret_cast<const f32x4*>(q + 64 + 4 * i);
        }
        // The product's value is the partials' sum rounded to bf16.
        unpack4(u32x2{pack2(a[0], a[1]), pack2(a[2], a[3])}, x);
        unpack4(u32x2{pack2(b[0], b[1]), pack2(b[2], b[3])}, x + 4);
    } else {
        unpack4(*reinterpret_cast<const u32x2*>(src + 4 * i), x);
        unpack4(*reinterpret_cast<const u32x2*>(src + 64 + 4 * i), x + 4);
    }
}

// cos and sin of position * inv_freq for lane i's four pairs: the angle in
// turns in 64 bits, whole turns taken off, then the hardware's sine and cosine
// of a turn's fraction.
__device__ __forceinline__ void angles(const AppendParams& P, int64_t pos, int i, float* cs, float* sn) {
    const f32x4 f = *reinterpret_cast<const f32x4*>(P.inv_freq + 4 * i);
    const double p = (double)pos * 0.15915494309189533577;  // / 2 pi
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const double turns = p * (double)f[j];
        const float frac = (float)(turns - rint(turns));
        cs[j] = __builtin_amdgcn_cosf(frac);
        sn[j] = __builtin_amdgcn_sinf(frac);
    }
}

// RMSNorm over the row's 16 lanes, then the rotation.
__device__ __forceinline__ void norm_rotate(float* x, const float* w, const float* cs, const float* sn, float eps) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(x[j], x[j], ss);
    ss += xor_desc<8>(ss);
    ss += xor_desc<4>(ss);
    ss += xor_desc<2>(ss);
    ss += xor_desc<1>(ss);
    const float rstd = rsqrtf(ss / (float)D + eps);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = x[j] * rstd * w[j], b = x[4 + j] * rstd * w[4 + j];
        x[j] = a * cs[j] - b * sn[j];
        x[4 + j] = b * cs[j] + a * sn[j];
    }
}

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;
}

// x * 2^-e as codes.  Only the largest exponent can leave a finite entry past 448.
__device__ __forceinline__ uint32_t quantise(const float* x, int e) {
    const float inv = pow2(-e);
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        y[j] = x[j] * inv;
        if (e == kMaxExp && fabsf(x[j]) < INFINITY) y[j] = fminf(fmaxf(y[j], -448.f), 448.f);
    }
    return codes4(y[0], y[1], y[2], y[3]);
}

// Four kept codes under a scale 2^d times finer (d = old - new <= 0).
__device__ __forceinline__ uint32_t rescale(uint32_t c, float f) {
    const float y0 = __builtin_amdgcn_cvt_f32_fp8((int)c, 0), y1 = __builtin_amdgcn_cvt_f32_fp8((int)c, 1);
    const float y2 = __builtin_amdgcn_cvt_f32_fp8((int)c, 2), y3 = __builtin_amdgcn_cvt_f32_fp8((int)c, 3);
    return codes4(y0 * f, y1 * f, y2 * f, y3 * f);
}

// NT threads take NT / 16 slots of a block at a time, IT times.
template <int NT, int IT, bool ROPE, bool PARTS>
__global__ __launch_bounds__(NT) void append_kernel(AppendParams P) {
    const int tid = threadIdx.x, i16 = tid & 15, row16 = tid >> 4;
    if constexpr (ROPE) {
        if ((int)blockIdx.x >= P.kv_groups) {
            // Queries: 16 lanes take q_heads heads of one token.
            const int chunks = (P.Hq + P.q_heads - 1) / P.q_heads;
            const int64_t g = (int64_t)((int)blockIdx.x - P.kv_groups) * (NT / 16) + row16;
            const bool live = g < (int64_t)P.T * chunks;
            const int t = live ? (int)(g / chunks) : 0, h0 = live ? (int)(g % chunks) * P.q_heads : 0;
            float cs[4], sn[4], w[8];
            angles(P, P.positions[t], i16, cs, sn);
            load_row<false>(P.qn, P, 0, i16, w);
            for (int j = 0; j < P.q_heads; ++j) {
                const int h = min(h0 + j, P.Hq - 1);
                const size_t e = ((size_t)t * (P.Hq + 2 * P.Hkv) + h) * D;
                float x[8];
                load_row<PARTS>(P.k + e, P, e, i16, x);
                norm_rotate(x, w, cs, sn, P.eps);
                if (live && h0 + j < P.Hq) {
                    uint16_t* dst = P.q_out + ((size_t)t * P.Hq + h) * D + 4 * i16;
                    *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(x[0], x[1]), pack2(x[2], x[3])};
                    *reinterpret_cast<u32x2*>(dst + 64) = u32x2{pack2(x[4], x[5]), pack2(x[6], x[7])};
                }
            }
            return;
        }
    }
    __shared__ int member[kMaxBlock];  // per slot of the block: the token that writes it, or -1
    __shared__ float red[2][NT / kWave];
    const int h = blockIdx.x % P.Hkv, t_first = blockIdx.x / P.Hkv * P.win;
    const int block = 1 << P.block_shift;
    for (int t = t_first; t < min(t_first + P.win, P.T); ++t) {  // uniform over the workgroup
        const int64_t slot = P.slots[t];
        if (slot < 0 || slot >= P.num_slots) continue;
        const int64_t blk = slot >> P.block_shift;
        const auto same = [&](int64_t s) { return s >= 0 && s < P.num_slots && (s >> P.block_shift) == blk; };
        if (t > 0 && same(P.slots[t - 1])) continue;
        int before = 0;
        for (int j = tid; j < t - 1; j += NT) before |= same(P.slots[j]);
        if (__syncthreads_or(before)) continue;  // an earlier token leads this block
        for (int j = tid; j < block; j += NT) member[j] = -1;
        __syncthreads();
        for (int j = t + tid; j < P.T; j += NT) {
            const int64_t s = P.slots[j];
            if (same(s)) atomicMax(&member[(int)(s & (block - 1))], j);
        }
        __syncthreads();
        // The block's place: head-major pages.
        const int64_t page = blk / (P.page_size >> P.block_shift);
        const int nb = (int)(blk - page * (P.page_size >> P.block_shift));
        const size_t row0 = ((size_t)page * P.Hkv + h) * P.page_size + (size_t)nb * block;
        const size_t sc = ((size_t)page * P.Hkv + h) * (P.page_size >> P.block_shift) + nb;
        const int old_k = min((int)P.k_scale[sc] - 127, kMaxExp), old_v = min((int)P.v_scale[sc] - 127, kMaxExp);
        float xk[IT][8], xv[IT][8];
        float ak = 0.f, av = 0.f;
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const int m = member[row16 + it * (NT / 16)], tm = max(m, 0);
            if constexpr (ROPE) {
                const size_t e = ((size_t)tm * (P.Hq + 2 * P.Hkv) + P.Hq + h) * D, ev = e + (size_t)P.Hkv * D;
                float cs[4], sn[4], w[8];
                load_row<PARTS>(P.k + e, P, e, i16, xk[it]);
                load_row<PARTS>(P.k + ev, P, ev, i16, xv[it]);
                angles(P, P.positions[tm], i16, cs, sn);
                load_row<false>(P.kn, P, 0, i16, w);
                norm_rotate(xk[it], w, cs, sn, P.eps);
            } else {
                load_row<false>(P.k + (size_t)tm * P.k_stride + (size_t)h * D, P, 0, i16, xk[it]);
                load_row<false>(P.v + (size_t)tm * P.v_stride + (size_t)h * D, P, 0, i16, xv[it]);
            }
            if (m >= 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    ak = fmaxf(ak, finite_abs(xk[it][j]));
                    av = fmaxf(av, finite_abs(xv[it][j]));
                }
            }
        }
        ak = wave_max(ak);
        av = wave_max(av);
        if ((tid & 63) == 0) {
            red[0][tid >> 6] = ak;
            red[1][tid >> 6] = av;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / kWave; ++w) {
            ak = fmaxf(ak, red[0][w]);
            av = fmaxf(av, red[1][w]);
        }
        const bool anew = member[0] >= 0;
        const int ek = anew ? need_exp(ak) : max(old_k, need_exp(ak));
        const int ev = anew ? need_exp(av) : max(old_v, need_exp(av));
        // Kept codes shrink by 2^(old - new): past 2^-20 nothing is left of 448.
        const float fk = pow2(max(old_k - ek, -20)), fv = pow2(max(old_v - ev, -20));
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const int r = row16 + it * (NT / 16);
            const int m = member[r];
            uint32_t* dk = reinterpret_cast<uint32_t*>(P.k_cache + (row0 + r) * D) + i16;
            uint32_t* dv = reinterpret_cast<uint32_t*>(P.v_cache + (row0 + r) * D) + i16;
            if (m >= 0) {
                dk[0] = quantise(xk[it], ek);
                dk[16] = quantise(xk[it] + 4, ek);
                dv[0] = quantise(xv[it], ev);
                dv[16] = quantise(xv[it] + 4, ev);
            } else if (anew) {
                dk[0] = dk[16] = dv[0] = dv[16] = 0u;
            } else {
                if (ek != old_k) {
                    const uint32_t a = dk[0], b = dk[16];
                    dk[0] = rescale(a, fk);
                    dk[16] = rescale(b, fk);
                }
                if (ev != old_v) {
                    const uint32_t a = dv[0], b = dv[16];
                    dv[0] = rescale(a, fv);
                    dv[16] = rescale(b, fv);
                }
            }
        }
        // Every thread has read the old scales before the last barrier.
        if (tid == 0) {
            P.k_scale[sc] = (uint8_t)(ek + 127);
            P.v_scale[sc] = (uint8_t)(ev + 127);
        }
        __syncthreads();  // member and red are used again
    }
}

template <int NT, int IT, bool ROPE, bool PARTS>
static int launch(AppendParams& P, hipStream_t s) {
    int64_t groups = P.kv_groups;
    if (ROPE) {
        const int64_t chunks = (P.Hq + P.q_heads - 1) / P.q_heads;
        groups += ((int64_t)P.T * chunks + NT / 16 - 1) / (NT / 16);
    }
    if (groups > (int64_t)UINT32_MAX / NT) return D3D_E_SHAPE;  // threads of a launch
    hipLaunchKernelGGL((append_kernel<NT, IT, ROPE, PARTS>), dim3((unsigned)groups), dim3(NT), 0, s, P);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? D3D_OK : (int)err;
}

template <bool ROPE, bool PARTS>
static int run(AppendParams& P, void* stream) {
    hipStream_t s = static_cast<hipStream_t>(stream);
    P.win = P.T > 1024 ? 16 : 1;
    P.q_heads = P.T > 1024 ? 8 : 1;
    const int64_t kv = ((int64_t)P.T + P.win - 1) / P.win * P.Hkv;
    if (kv > INT_MAX) return D3D_E_SHAPE;
    P.kv_groups = (int)kv;
    switch (P.block_shift) {
        case 4: return launch<256, 1, ROPE, PARTS>(P, s);
        case 5: return launch<512, 1, ROPE, PARTS>(P, s);
        case 6: return launch<1024, 1, ROPE, PARTS>(P, s);
        case 7: return launch<1024, 2, ROPE, PARTS>(P, s);
        default: return launch<1024, 4, ROPE, PARTS>(P, s);
    }
}

static bool off(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

// The cache's part of the arguments.
static int cache_args(AppendParams& P, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                      const int64_t* slots, int T, int Hkv, int D_, int page_size, int block, int num_pages) {
    if (T < 0 || Hkv < 1 || page_size < 1 || num_pages < 1) return D3D_E_SHAPE;
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
    P.k = static_cast<const uint16_t*>(qkv);
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
