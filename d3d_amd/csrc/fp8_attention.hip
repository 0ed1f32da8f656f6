// Paged block attention over the 8-bit cache (fp8_cache.hpp): causal blocks
// (verify, prefill slices, single tokens), bidirectional blocks (draft) and
// packed multi-branch blocks, with the visibility rules of the bf16 forms
// (attention.hip).
//
// One wave per (request, query, query head).  Lanes take tokens of a chunk of
// 64 for the scores, then two output dimensions each for the weighted sum of
// the values; the softmax runs online over the chunks, in fp32.
#include "fp8_cache.hpp"
#include "../../include/d3d_hip.h"

#include <limits.h>

namespace d3d {
namespace fp8 {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct AttnParams {
    const uint16_t* q;
    const uint8_t* k_cache;
    const uint8_t* v_cache;
    const uint8_t* k_scale;
    const uint8_t* v_scale;
    const int32_t* block_table;
    const int32_t* context_lens;
    const int32_t* vis;
    uint16_t* out;
    int B, Q, Hq, Hkv, G;
    int page_size, block_shift, max_pages, num_pages;
    int max_context;
    float scale_log2;
};

enum : int { kCausal = 0, kFull = 1, kPacked = 2 };

template <int MODE>
__global__ __launch_bounds__(256) void attn_kernel(AttnParams P) {
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (int64_t)P.B * P.Q * P.Hq) return;  // whole wave; no barrier in this kernel
    const int h = (int)(id % P.Hq), i = (int)(id / P.Hq % P.Q), b = (int)(id / P.Hq / P.Q);
    const int kvh = h / P.G;
    const int ctx = min(P.context_lens[b], P.max_pages * P.page_size);
    int va = ctx, lo = 0, hi = 0;
    if (MODE == kCausal) va = ctx - P.Q + i + 1;
    if (MODE == kPacked) {
        va = ctx - P.Q + P.vis[3 * i];
        lo = ctx - P.Q + P.vis[3 * i + 1];
        hi = ctx - P.Q + P.vis[3 * i + 2];
    }
    const int end = min(min(ctx, P.max_context), max(va, MODE == kPacked ? hi : va));
    const uint16_t* q = P.q + id * D;
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    const int nb = P.page_size >> P.block_shift;
    for (int t0 = 0; t0 < end; t0 += 64) {
        const int t = t0 + lane;
        const bool seen = t < end && (t < va || (MODE == kPacked && t >= lo && t < hi));
        size_t row = 0;
        float vs = 0.f, s = -INFINITY;
        bool has = false;
        if (seen) {
            const int page = P.block_table[(size_t)b * P.max_pages + t / P.page_size], in = t % P.page_size;
            has = page >= 0 && page < P.num_pages;
            float dot = 0.f;
            if (has) {
                const size_t ph = (size_t)page * P.Hkv + kvh, sc = ph * nb + (in >> P.block_shift);
                row = ph * P.page_size + in;
                const uint32_t* k = reinterpret_cast<const uint32_t*>(P.k_cache + row * D);
                for (int d = 0; d < D / 4; ++d) {
                    const int w = (int)k[d];
                    dot += bf16_bits_to_f32(q[4 * d]) * __builtin_amdgcn_cvt_f32_fp8(w, 0);
                    dot += bf16_bits_to_f32(q[4 * d + 1]) * __builtin_amdgcn_cvt_f32_fp8(w, 1);
                    dot += bf16_bits_to_f32(q[4 * d + 2]) * __builtin_amdgcn_cvt_f32_fp8(w, 2);
                    dot += bf16_bits_to_f32(q[4 * d + 3]) * __builtin_amdgcn_cvt_f32_fp8(w, 3);
                }
                dot *= exp2f((float)((int)P.k_scale[sc] - 127));
                vs = exp2f((float)((int)P.v_scale[sc] - 127));
            }
            s = dot * P.scale_log2;  // a page outside the pool reads as zeros
        }
        const float m_new = fmaxf(m, wave_max(s));
        const float off = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = m == -INFINITY ? 0.f : exp2f(m - off);
        const float p = seen ? exp2f(s - off) : 0.f;
        l = l * alpha + wave_sum(p);
        o0 *= alpha;
        o1 *= alpha;
        m = m_new;
        const float pv = p * vs;
        for (int j = 0; j < 64; ++j) {
            const float w = __shfl(pv, j, 64);
            const size_t r = (size_t)__shfl((unsigned long long)row, j, 64);
            if (!__shfl((int)has, j, 64)) continue;  // keys that this row does not see take no part
            const int c = (int)*reinterpret_cast<const uint16_t*>(P.v_cache + r * D + 2 * lane);
            o0 += w * __builtin_amdgcn_cvt_f32_fp8(c, 0);
            o1 += w * __builtin_amdgcn_cvt_f32_fp8(c, 1);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* out = P.out + id * D + 2 * lane;
    out[0] = f32_to_bf16_bits(o0 * inv);
    out[1] = f32_to_bf16_bits(o1 * inv);
}

template <int MODE>
static int attn_run(const void* q, const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                    const int32_t* block_table, const int32_t* context_lens, const int32_t* vis, void* out, int B,
                    int Q, int Hq, int Hkv, int D_, int page_size, int block, int max_pages, int num_pages,
                    float scale, int max_context, void* workspace, size_t ws_bytes, void* stream) {
    if (B < 1 || B > 65535 || Q < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv) return D3D_E_SHAPE;
    if (D_ != D || Hq / Hkv > 64) return D3D_E_UNSUPPORTED;
    if (page_size < 1 || max_pages < 1 || num_pages < 1 || max_context < 1) return D3D_E_SHAPE;
    if ((int64_t)max_pages * page_size > INT_MAX || (int64_t)max_pages * page_size < max_context) return D3D_E_SHAPE;
    const int sh = fp8_block_shift(page_size, block);
    if (sh < 0) return D3D_E_UNSUPPORTED;
    if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !block_table || !context_lens || !out) return D3D_E_NULL;
    if (MODE == kPacked && !vis) return D3D_E_NULL;
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16)
        return D3D_E_UNSUPPORTED;
    AttnParams P;
    P.q = static_cast<const uint16_t*>(q);
    P.k_cache = static_cast<const uint8_t*>(k_cache);
    P.v_cache = static_cast<const uint8_t*>(v_cache);
    P.k_scale = static_cast<const uint8_t*>(k_scale);
    P.v_scale = static_cast<const uint8_t*>(v_scale);
    P.block_table = block_table;
    P.context_lens = context_lens;
    P.vis = vis;
    P.out = static_cast<uint16_t*>(out);
    P.B = B;
    P.Q = Q;
    P.Hq = Hq;
    P.Hkv = Hkv;
    P.G = Hq / Hkv;
    P.page_size = page_size;
    P.block_shift = sh;
    P.max_pages = max_pages;
    P.num_pages = num_pages;
    P.max_context = max_context;
    P.scale_log2 = scale * 1.4426950408889634f;
    const int64_t groups = ((int64_t)B * Q * Hq + 3) / 4;
    if (groups > (int64_t)UINT32_MAX / 256) return D3D_E_SHAPE;
    hipLaunchKernelGGL((attn_kernel<MODE>), dim3((unsigned)groups), dim3(256), 0, static_cast<hipStream_t>(stream), P);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? D3D_OK : (int)err;
}

}  // namespace fp8
}  // namespace d3d

using namespace d3d;

extern "C" size_t d3d_attn_fp8_workspace_bytes(int B, int Q, int Hq, int Hkv, int D, int page_size, int max_context) {
    if (B < 1 || Q < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || D != fp8::D || page_size < 1 || max_context < 1) return 0;
    return 256;
}

extern "C" int d3d_verify_attn_paged_fp8(const void* q, const void* k_cache, const void* v_cache, const void* k_scale,
                                         const void* v_scale, const int32_t* block_table, const int32_t* context_lens,
                                         void* out, int B, int Q, int Hq, int Hkv, int D, int page_size, int block,
                                         int max_pages, int num_pages, float scale, int max_context, void* workspace,
                                         size_t workspace_bytes, void* stream) {
    return fp8::attn_run<fp8::kCausal>(q, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, nullptr, out,
                                       B, Q, Hq, Hkv, D, page_size, block, max_pages, num_pages, scale, max_context,
                                       workspace, workspace_bytes, stream);
}

extern "C" int d3d_draft_block_attn_fp8(const void* q, const void* k_cache, const void* v_cache, const void* k_scale,
                                        const void* v_scale, const int32_t* block_table, const int32_t* context_lens,
                                        void* out, int B, int Q, int Hq, int Hkv, int D, int page_size, int block,
                                        int max_pages, int num_pages, float scale, int max_context, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    return fp8::attn_run<fp8::kFull>(q, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, nullptr, out, B,
                                     Q, Hq, Hkv, D, page_size, block, max_pages, num_pages, scale, max_context,
                                     workspace, workspace_bytes, stream);
}

extern "C" int d3d_packed_block_attn_fp8(const void* q, const void* k_cache, const void* v_cache, const void* k_scale,
                                         const void* v_scale, const int32_t* block_table, const int32_t* context_lens,
                                         const int32_t* q_visibility, void* out, int B, int Q, int Hq, int Hkv, int D,
                                         int page_size, int block, int max_pages, int num_pages, float scale,
                                         int max_context, void* workspace, size_t workspace_bytes, void* stream) {
    return fp8::attn_run<fp8::kPacked>(q, k_cache, v_cache, k_scale, v_scale, block_table, context_lens, q_visibility,
                                       out, B, Q, Hq, Hkv, D, page_size, block, max_pages, num_pages, scale,
                                       max_context, workspace, workspace_bytes, stream);
}
