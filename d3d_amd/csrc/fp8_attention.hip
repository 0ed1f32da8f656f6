// Paged block attention over the 8-bit cache (fp8_cache.hpp): causal blocks
// (verify, prefill slices, single tokens), bidirectional blocks (draft) and
// packed multi-branch blocks, with the visibility rules of the bf16 forms
// (attention.hip).
//
// Work: a workgroup takes (request, KV head, up to 64 rows = query heads of the
// group x queries, a range of the context), its waves take the range's 32-token
// steps in turn.  A wave holds all of the workgroup's rows, so each key and
// value is fetched, converted and multiplied by one wave only: keys go from
// memory to registers, values through the wave's own LDS rows to be
// transposed, and the main loop has no barrier.  (Waves that share a staged
// tile and split the rows instead, as the bf16 kernel's do, would each read
// and convert every key and value again.)
//
// Scores are computed transposed, S^T = K Q^T, with v_mfma_f32_16x16x32_bf16 on
// the keys converted with their scale (exact): lane l holds tokens 4 (l / 16) +
// r of row l % 16, which two 16-token groups at a time is the operand layout of
// P^T in O^T = V^T P^T.  The row maximum that probabilities are taken against
// moves only when a score passes it by 2^8: until then no lane talks to
// another and no accumulator is rescaled.  At the end the waves' (m, l, O) are
// merged through LDS; with more than one range per request partial results go
// to the workspace and a second launch merges them.
#include "fp8_cache.hpp"
#include "../../include/d3d_hip.h"

#include <limits.h>

#include <algorithm>

namespace d3d {
namespace fp8 {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 32;       // tokens a wave takes at a time
constexpr int kTile = 128;      // tokens four waves take at a time: the unit of ranges
constexpr int kMaxTiles = 64;   // tiles of a range whose pages and scales are staged at once
constexpr int kVRow = D + 16;   // LDS bytes per value row: 16 rows, 36 banks apart, read without conflicts
constexpr float kLazy = 8.f;    // how far (log2) scores may pass the maximum that they are taken against

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
    _Float16* part_o;  // [item][nqt][Hkv][M][D], O / l of a range, times 2^-e
    f32x4* part_ml;    // [item][nqt][Hkv][M]: m, l, 2^e of dims 0..63, of 64..127
    int B, Q, Hq, Hkv, G, QT, nqt, M;
    int page_size, block_shift, max_pages, num_pages;
    int max_context;
    int items;   // ranges of all requests at most
    int slots;   // workgroups that run at once
    int min_tiles;  // tiles per range at least
    int dense;   // ranges per request when items are not packed (B > 64), else 0
    int dense_tiles;
    float scale_log2;
};

enum : int { kCausal = 0, kFull = 1, kPacked = 2 };

__device__ __forceinline__ int ctx_of(const AttnParams& P, int b) {
    return min(P.context_lens[b], min(P.max_pages * P.page_size, P.max_context));
}

__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// How the context is cut, the same in every workgroup of both launches.  Up to
// 64 requests: ranges of `tiles` whole tiles, the least number of tiles that
// keeps the ranges of all requests within P.slots workgroups; item numbers
// run through the requests' own range counts.  A whole wave calls it.
struct Range {
    int b, s, n, tiles, first;  // request (-1: none), range, ranges of the request, tiles per range, its first item
};

__device__ __forceinline__ void cut_of(const AttnParams& P, int lane, int& tiles, int& incl, int& n) {
    const int t = lane < P.B ? (max(ctx_of(P, lane), 1) + kTile - 1) / kTile : 0;
    const int per = P.Hkv * P.nqt, room = max(P.slots / per, 1);
    const int total = wave_sum_int(t);
    tiles = max(P.min_tiles, (total + room - 1) / room);
    for (;;) {
        n = lane < P.B ? (t + tiles - 1) / tiles : 0;
        const int sum = wave_sum_int(n);
        if (sum <= max(room, P.B)) break;  // one range each at the least
        tiles += max(1, tiles * (sum - room) / (2 * sum));
    }
    incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(incl, o, 64);
        if (lane >= o) incl += u;
    }
}

__device__ __forceinline__ Range range_of_item(const AttnParams& P, int item) {
    Range r;
    if (P.dense) {
        r.b = P.B - 1 - item / P.dense;  // later requests first: a prompt's longer slices
        r.s = item % P.dense;
        r.tiles = P.dense_tiles;
        r.n = max(1, (ctx_of(P, r.b) + kTile * r.tiles - 1) / (kTile * r.tiles));
        r.first = item - r.s;
        if (r.s >= r.n) r.b = -1;
        return r;
    }
    const int lane = threadIdx.x & 63;
    int incl, n;
    cut_of(P, lane, r.tiles, incl, n);
    const uint64_t past = __ballot(lane < P.B && incl > item);
    if (!past) {
        r.b = -1;
        r.s = r.n = r.first = 0;
        return r;
    }
    r.b = __builtin_ctzll(past);
    r.n = __shfl(n, r.b, 64);
    r.first = __shfl(incl, r.b, 64) - r.n;
    r.s = item - r.first;
    return r;
}

__device__ __forceinline__ Range range_of_request(const AttnParams& P, int b) {
    Range r;
    r.b = b;
    r.s = 0;
    if (P.dense) {
        r.tiles = P.dense_tiles;
        r.n = max(1, (ctx_of(P, b) + kTile * r.tiles - 1) / (kTile * r.tiles));
        r.first = (P.B - 1 - b) * P.dense;
        return r;
    }
    const int lane = threadIdx.x & 63;
    int incl, n;
    cut_of(P, lane, r.tiles, incl, n);
    r.n = __shfl(n, b, 64);
    r.first = __shfl(incl, b, 64) - r.n;
    return r;
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    const f32x2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// Eight codes with their scale as an MFMA operand.
__device__ __forceinline__ bf16x8 widen8(uint32_t a, uint32_t b, float sa, float sb) {
    const bf16x2 w[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sa, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sa, true),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sb, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sb, true)};
    return bf16x8{w[0][0], w[0][1], w[1][0], w[1][1], w[2][0], w[2][1], w[3][0], w[3][1]};
}

// Eight rows of 16 codes transposed (ds_read_b64_tr_b8): lane i of 16 gives the
// address of row i / 2, columns 8 (i % 2) .. + 7, and gets column i of the rows.
__device__ __forceinline__ u32x2 lds_read_tr8(const char* p) {
    return __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(const __attribute__((address_space(3))) char*)p));
}

__device__ __forceinline__ float across_max(float v) {
    v = fmaxf(v, xor_desc<32>(v));
    return fmaxf(v, xor_desc<16>(v));
}
__device__ __forceinline__ float across_sum(float v) {
    v += xor_desc<32>(v);
    return v + xor_desc<16>(v);
}

// Bytes that are NaN codes, as a mask of 0xff.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
    const uint32_t hit = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return (hit >> 7) * 0xffu;
}

template <int MODE, int RT, int NW>
__global__ __launch_bounds__(NW * 64, RT == 4 ? 1 : 2) void attn_kernel(AttnParams P) {
    constexpr int NT = NW * 64, R = 16 * RT;
    constexpr int kGroups = kMaxTiles * kTile / 16;
    // Output exchange: half the dimensions at a time, a row's floats padded.
    constexpr int kHalf = D / 2, kORow = kHalf + 4;
    constexpr int kVBytes = NW * kStep * kVRow, kOBytes = NW * R * kORow * 4;
    __shared__ __attribute__((aligned(16))) char lds[kVBytes > kOBytes ? kVBytes : kOBytes];
    __shared__ int row_of[kGroups];       // first cache row of a 16-token group, -1: no page
    __shared__ u32x2 scale_of[kGroups];   // its key and value scales
    __shared__ float stat[2][NW][R];

    const int kvh = blockIdx.x % P.Hkv, qt = blockIdx.y, item = blockIdx.x / P.Hkv;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int g4 = lane >> 4, c16 = lane & 15;
    const Range rg = range_of_item(P, item);
    const int b = __builtin_amdgcn_readfirstlane(rg.b);
    if (b < 0) return;  // uniform, before any barrier
    const int ctx = ctx_of(P, b), q0 = qt * P.QT;
    const int t_begin = __builtin_amdgcn_readfirstlane(rg.s) * __builtin_amdgcn_readfirstlane(rg.tiles) * kTile;

    // This lane's rows: head gh of the group, query qi; visible keys t < va, vlo <= t < vhi.
    int qi[RT], head[RT], va[RT], vlo[RT], vhi[RT];
    bool row_ok[RT];
    int a_min = INT_MAX, a_max = 0, s_lo = INT_MAX, s_hi = 0;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = rt * 16 + c16, gh = row / P.QT;
        qi[rt] = q0 + row - gh * P.QT;
        row_ok[rt] = row < P.M && qi[rt] < P.Q;
        head[rt] = kvh * P.G + (row_ok[rt] ? gh : 0);
        va[rt] = vlo[rt] = vhi[rt] = 0;
        if (row_ok[rt]) {
            // The frontier goes by the context's own length, reads by its bounds.
            const int pre = min(P.context_lens[b], P.max_pages * P.page_size) - P.Q;
            va[rt] = ctx;
            if constexpr (MODE == kCausal) va[rt] = pre + qi[rt] + 1;
            if constexpr (MODE == kPacked) {
                va[rt] = pre + P.vis[qi[rt] * 3];
                vlo[rt] = max(pre + P.vis[qi[rt] * 3 + 1], 0);
                vhi[rt] = min(pre + P.vis[qi[rt] * 3 + 2], ctx);
            }
            va[rt] = min(va[rt], ctx);
            a_min = min(a_min, va[rt]);
            a_max = max(a_max, va[rt]);
            if (MODE == kPacked && vlo[rt] < vhi[rt]) {
                s_lo = min(s_lo, vlo[rt]);
                s_hi = max(s_hi, vhi[rt]);
            }
        }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        a_min = min(a_min, __shfl_xor(a_min, o, 64));
        a_max = max(a_max, __shfl_xor(a_max, o, 64));
        if constexpr (MODE == kPacked) {
            s_lo = min(s_lo, __shfl_xor(s_lo, o, 64));
            s_hi = max(s_hi, __shfl_xor(s_hi, o, 64));
        }
    }
    a_min = __builtin_amdgcn_readfirstlane(a_min);
    a_max = __builtin_amdgcn_readfirstlane(a_max);
    s_lo = __builtin_amdgcn_readfirstlane(s_lo);
    s_hi = __builtin_amdgcn_readfirstlane(s_hi);
    const int t_last = min(t_begin + __builtin_amdgcn_readfirstlane(rg.tiles) * kTile, ctx);

    // Q^T operands: dims 64 p + 16 g4 + 8 e .. + 7 at ks = 2 p + e, as the keys are loaded.
    bf16x8 qop[RT][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            u32x4 v = {0u, 0u, 0u, 0u};
            if (row_ok[rt])
                v = *reinterpret_cast<const u32x4*>(P.q + (((size_t)b * P.Q + qi[rt]) * P.Hq + head[rt]) * D +
                                                    64 * (ks >> 1) + 16 * g4 + 8 * (ks & 1));
            qop[rt][ks] = __builtin_bit_cast(bf16x8, v);
        }

    f32x4 o[RT][8];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int n = 0; n < 8; ++n) o[rt][n] = {0.f, 0.f, 0.f, 0.f};
        m[rt] = -INFINITY;
        l[rt] = 0.f;
    }

    char* vbuf = lds + w * (kStep * kVRow);
    // The value row that this lane stores: token j 8 + lane / 8 goes to row 8 g +
    // 4 sub + r (token 16 sub + 4 g + r), so that a group's eight are neighbours.
    const int vt = lane >> 3;  // token within 8
    const auto vrow = [&](int tok) { return 8 * ((tok >> 2) & 3) + 4 * (tok >> 4) + (tok & 3); };
    const uint32_t k_off = (uint32_t)(c16 * D + 16 * g4);
    const uint32_t v_off = (uint32_t)(vt * D + 16 * (lane & 7));

    // The range in pieces of at most kMaxTiles tiles whose pages and scales fit the tables.
    for (int p0 = t_begin; p0 < t_last; p0 += kMaxTiles * kTile) {
        const int p_end = min(p0 + kMaxTiles * kTile, t_last);
        // Steps that some row sees: those below a_max, then those of [s_lo, s_hi).
        const int n1 = max(0, (min(a_max, p_end) - p0 + kStep - 1) / kStep);
        int st2 = n1, n2 = 0;
        if constexpr (MODE == kPacked) {
            if (s_lo < s_hi) {
                st2 = max(n1, (s_lo - p0) / kStep);
                n2 = max(0, (min(s_hi, p_end) - p0 + kStep - 1) / kStep - st2);
            }
        }
        const int steps = n1 + n2;
        if (steps == 0) continue;
        const auto step_at = [&](int j) { return j < n1 ? j : st2 + j - n1; };
        __syncthreads();  // the tables of the piece before are no longer read
        const int groups = 2 * (step_at(steps - 1) + 1);
        for (int i = threadIdx.x; i < groups; i += NT) {
            const int t = p0 + 16 * i;
            int row = -1;
            u32x2 sc = {0x3f800000u, 0x3f800000u};
            if (t < p_end) {
                const int pi = t / P.page_size, in = t - pi * P.page_size;
                const int page = P.block_table[(size_t)b * P.max_pages + pi];
                if (page >= 0 && page < P.num_pages) {
                    const size_t ph = (size_t)page * P.Hkv + kvh;
                    const size_t at = ph * (P.page_size >> P.block_shift) + (in >> P.block_shift);
                    row = (int)(ph * P.page_size + in);
                    sc[0] = (uint32_t)P.k_scale[at] << 23;
                    sc[1] = (uint32_t)P.v_scale[at] << 23;
                }
            }
            row_of[i] = row;
            scale_of[i] = sc;
        }
        __syncthreads();

        u32x4 kr[2][2], vr[4];
        const auto fetch = [&](int j) {
            const int g = 2 * step_at(j);
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const int row = max(__builtin_amdgcn_readfirstlane(row_of[g + sub]), 0);
                const uint8_t* kb = P.k_cache + (size_t)row * D;
                const uint8_t* vb = P.v_cache + (size_t)row * D;
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    kr[sub][p] = *reinterpret_cast<const u32x4*>(kb + k_off + 64 * p);
                    vr[2 * sub + p] = *reinterpret_cast<const u32x4*>(vb + v_off + 8 * D * p);
                }
            }
        };
        if (w < steps) fetch(w);
        for (int j = w; j < steps; j += NW) {
            const int t0 = p0 + kStep * step_at(j), g = 2 * step_at(j);
            const bool ok0 = __builtin_amdgcn_readfirstlane(row_of[g]) >= 0;
            const bool ok1 = __builtin_amdgcn_readfirstlane(row_of[g + 1]) >= 0;
            // Keys that some row does not see, or no page: the uncommon step.
            const bool edge = t0 + kStep > min(a_min, p_end) || !ok0 || !ok1;
            const float ks0 = __uint_as_float(__builtin_amdgcn_readfirstlane(scale_of[g][0]));
            const float vs0 = __uint_as_float(__builtin_amdgcn_readfirstlane(scale_of[g][1]));
            const float ks1 = __uint_as_float(__builtin_amdgcn_readfirstlane(scale_of[g + 1][0]));
            const float vs1 = __uint_as_float(__builtin_amdgcn_readfirstlane(scale_of[g + 1][1]));
            bool poison = false;
            if (edge) {
                // Values that no row may see become 0, and NaN values, which a
                // probability of 0 would not keep out, are put in at the end.
                bool bad = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = 8 * i + vt;
                    const bool keep = t0 + tok < p_end && (i < 2 ? ok0 : ok1);
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const uint32_t c = keep ? vr[i][d] : 0u, nb = nan_bytes(c);
                        bad |= nb != 0;
                        vr[i][d] = c & ~nb;
                    }
                }
                poison = __any(bad);
                if (!ok0) kr[0][0] = kr[0][1] = u32x4{0u, 0u, 0u, 0u};
                if (!ok1) kr[1][0] = kr[1][1] = u32x4{0u, 0u, 0u, 0u};
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<u32x4*>(vbuf + vrow(8 * i + vt) * kVRow + 16 * (lane & 7)) = vr[i];
            bf16x8 kf[2][4];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                kf[0][2 * p] = widen8(kr[0][p][0], kr[0][p][1], ks0, ks0);
                kf[0][2 * p + 1] = widen8(kr[0][p][2], kr[0][p][3], ks0, ks0);
                kf[1][2 * p] = widen8(kr[1][p][0], kr[1][p][1], ks1, ks1);
                kf[1][2 * p + 1] = widen8(kr[1][p][2], kr[1][p][3], ks1, ks1);
            }
            if (j + NW < steps) fetch(j + NW);

            // sc[rt][sub][r]: token t0 + 16 sub + 4 g4 + r, row c16 of row tile rt.
            f32x4 sc[RT][2];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sc[rt][0] = sc[rt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        sc[rt][sub] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[sub][ks], qop[rt][ks], sc[rt][sub], 0, 0, 0);
            if (edge) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int t = t0 + 16 * sub + 4 * g4 + r;
                            const bool seen = t < va[rt] || (MODE == kPacked && t >= vlo[rt] && t < vhi[rt]);
                            if (!(seen && t < p_end)) sc[rt][sub][r] = -INFINITY;
                        }
            }
            // Scores (log2) past a row's reference by kLazy move it, for all lanes of the row.
            bool grow = false;
            float top[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float t = fmaxf(sc[rt][0][0], sc[rt][0][1]);
                t = fmaxf(fmaxf(t, sc[rt][0][2]), sc[rt][0][3]);
                t = fmaxf(fmaxf(t, sc[rt][1][0]), sc[rt][1][1]);
                t = fmaxf(fmaxf(t, sc[rt][1][2]), sc[rt][1][3]);
                top[rt] = t * P.scale_log2;
                grow |= top[rt] > m[rt] + kLazy;
            }
            if (__any(grow)) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const float mn = fmaxf(m[rt], across_max(top[rt]));
                    const float alpha = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rt] - mn);
                    l[rt] *= alpha;
#pragma unroll
                    for (int n = 0; n < 8; ++n) o[rt][n] *= alpha;
                    m[rt] = mn;
                }
            }
            bf16x8 pop[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float off = m[rt] == -INFINITY ? 0.f : m[rt];
                float p[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[rt][i >> 2][i & 3], P.scale_log2, -off));
                    l[rt] += p[i];
                }
                pop[rt] = __builtin_bit_cast(bf16x8, u32x4{pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]),
                                                           pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])});
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const u32x2 c = lds_read_tr8(vbuf + (8 * g4 + (c16 >> 1)) * kVRow + 16 * n + 8 * (c16 & 1));
                const bf16x8 vf = widen8(c[0], c[1], vs0, vs1);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    o[rt][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pop[rt], o[rt][n], 0, 0, 0);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (poison) {
                // Rows that see a NaN value: its dimension is NaN.
                for (int tok = 0; tok < kStep; ++tok) {
                    const int t = t0 + tok, row = row_of[g + (tok >> 4)];
                    if (t >= p_end || row < 0) continue;
                    const uint32_t* src = reinterpret_cast<const uint32_t*>(P.v_cache + ((size_t)row + (tok & 15)) * D) + g4;
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const uint32_t nb = nan_bytes(src[4 * n]);
                        if (!nb) continue;
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            const bool seen = t < va[rt] || (MODE == kPacked && t >= vlo[rt] && t < vhi[rt]);
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (seen && ((nb >> (8 * r)) & 1)) o[rt][n][r] = NAN;
                        }
                    }
                }
            }
        }
    }

    // The waves' statistics, then their sums, half the dimensions at a time.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] = across_sum(l[rt]);
        if (g4 == 0) {
            stat[0][w][16 * rt + c16] = m[rt];
            stat[1][w][16 * rt + c16] = l[rt];
        }
    }
    __syncthreads();  // also: no wave reads its value rows any more
    float mx[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        mx[rt] = -INFINITY;
#pragma unroll
        for (int v = 0; v < NW; ++v) mx[rt] = fmaxf(mx[rt], stat[0][v][16 * rt + c16]);
        const float f = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rt] - mx[rt]);
#pragma unroll
        for (int n = 0; n < 8; ++n) o[rt][n] *= f;
    }
    // Thread tid adds up dims dp .. of row tr; TPR threads per row.
    constexpr int TPR = NT / R, DPT = kHalf / TPR;
    static_assert(TPR >= 1 && TPR <= 64 && DPT >= 1, "threads per row");
    const int tr = threadIdx.x / TPR, dp = (threadIdx.x % TPR) * DPT;
    float rm = -INFINITY, rl = 0.f;
#pragma unroll
    for (int v = 0; v < NW; ++v) rm = fmaxf(rm, stat[0][v][tr]);
#pragma unroll
    for (int v = 0; v < NW; ++v) {
        const float mv = stat[0][v][tr];
        rl += (mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mv - rm)) * stat[1][v][tr];
    }
    const float inv = rl == 0.f ? 0.f : 1.f / rl;
    const int orow_h = tr / P.QT, orow_q = q0 + tr - orow_h * P.QT;
    const bool live = tr < P.M && orow_q < P.Q;
    const size_t unit = ((size_t)item * P.nqt + qt) * P.Hkv + kvh;
    float es[2];
    float* ex = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (half) __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int n = 0; n < 4; ++n)
                *reinterpret_cast<f32x4*>(ex + (size_t)(w * R + 16 * rt + c16) * kORow + 16 * n + 4 * g4) = o[rt][4 * half + n];
        __syncthreads();
        float sum[DPT];
#pragma unroll
        for (int d = 0; d < DPT; ++d) {
            sum[d] = 0.f;
#pragma unroll
            for (int v = 0; v < NW; ++v) sum[d] += ex[(size_t)(v * R + tr) * kORow + dp + d];
            sum[d] *= inv;
        }
        if (rg.n == 1) {
            if (live) {
                uint16_t* dst = P.out + (((size_t)b * P.Q + orow_q) * P.Hq + kvh * P.G + orow_h) * D + kHalf * half + dp;
                if constexpr (DPT % 2 == 0) {
#pragma unroll
                    for (int d = 0; d < DPT; d += 2)
                        *reinterpret_cast<uint32_t*>(dst + d) = pack_bf16x2(sum[d], sum[d + 1]);
                } else {
#pragma unroll
                    for (int d = 0; d < DPT; ++d) dst[d] = f32_to_bf16_bits(sum[d]);
                }
            }
        } else {
            // fp16 with a power of two per row and half: the largest lands in
            // [2^14, 2^15), so nothing overflows and 2^-12 of it is kept.
            float amax = 0.f;
#pragma unroll
            for (int d = 0; d < DPT; ++d) amax = fmaxf(amax, fabsf(sum[d]));
#pragma unroll
            for (int s = 1; s < TPR; s <<= 1) amax = fmaxf(amax, __shfl_xor(amax, s, 64));
            const int e = min(max((int)((__float_as_uint(amax) >> 23) & 0xffu) - 127 - 14, -110), 110);
            es[half] = pow2(e);
            if (tr < P.M) {
                _Float16* dst = P.part_o + (unit * P.M + tr) * D + kHalf * half + dp;
#pragma unroll
                for (int d = 0; d < DPT; ++d) dst[d] = (_Float16)(sum[d] * pow2(-e));
            }
        }
    }
    if (rg.n > 1 && tr < P.M && threadIdx.x % TPR == 0) P.part_ml[unit * P.M + tr] = f32x4{rm, rl, es[0], es[1]};
}

// Merges the ranges of a request: workgroup (8 rows, KV head, request and
// query tile), 32 threads per row, 4 dims each.
constexpr int kRows = 8, kMaxRanges = 512;

__global__ __launch_bounds__(256) void attn_merge_kernel(AttnParams P) {
    const int b = blockIdx.z / P.nqt, qt = blockIdx.z - b * P.nqt, kvh = blockIdx.y;
    const Range rg = range_of_request(P, b);
    if (rg.n == 1) return;  // written by the first launch
    __shared__ float wt[kRows][kMaxRanges];
    const int rr = threadIdx.x / 32, c4 = (threadIdx.x % 32) * 4, row = blockIdx.x * kRows + rr;
    const int row_c = min(row, P.M - 1), l32 = threadIdx.x & 31;
    const auto unit = [&](int s) { return (((size_t)(rg.first + s) * P.nqt + qt) * P.Hkv + kvh) * P.M + row_c; };
    float mx = -INFINITY;
    for (int s = l32; s < rg.n; s += 32) mx = fmaxf(mx, P.part_ml[unit(s)][0]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    float den = 0.f;
    for (int s = l32; s < rg.n; s += 32) {
        const f32x4 ml = P.part_ml[unit(s)];
        const float wgt = (ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - mx)) * ml[1];
        den += wgt;
        wt[rr][s] = wgt;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) den += __shfl_xor(den, o, 64);
    __syncthreads();
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < rg.n; ++s) {
        const size_t u = unit(s);
        const float f = wt[rr][s] * P.part_ml[u][2 + (c4 >> 6)];
        const h16x4 h = *reinterpret_cast<const h16x4*>(P.part_o + u * D + c4);
        acc += f * f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    const int gh = row / P.QT, q = qt * P.QT + row - gh * P.QT;
    if (row >= P.M || q >= P.Q) return;
    *reinterpret_cast<u32x2*>(P.out + (((size_t)b * P.Q + q) * P.Hq + kvh * P.G + gh) * D + c4) =
        u32x2{pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
}

struct AttnPlan {
    int QT, nqt, M, rt, items, slots, min_tiles, dense, dense_tiles;
    bool merge;
    size_t o_bytes, bytes;
};

static AttnPlan attn_plan(int B, int Q, int Hq, int Hkv, int max_context) {
    AttnPlan p{};
    const int G = Hq / Hkv;
    p.QT = std::min(Q, 64 / G);
    p.nqt = (Q + p.QT - 1) / p.QT;
    p.M = G * p.QT;
    p.rt = p.M <= 16 ? 1 : p.M <= 32 ? 2 : 4;
    p.slots = p.rt == 4 ? 256 : 512;
    p.min_tiles = 2;
    const int64_t units = (int64_t)Hkv * p.nqt;
    const int tiles = (max_context + kTile - 1) / kTile;
    if (B <= 64) {
        const int room = (int)std::max<int64_t>(p.slots / units, 1);
        p.items = std::max(B, room);
        const int64_t most = (int64_t)B * ((tiles + p.min_tiles - 1) / p.min_tiles);
        p.items = (int)std::min<int64_t>(p.items, std::max<int64_t>(most, 1));
        p.merge = p.items > B || (B > 1 && tiles > p.min_tiles);
    } else {
        p.dense = (int)std::max<int64_t>(1, std::min<int64_t>(4096 / (units * B), kMaxRanges));
        p.dense_tiles = std::max((tiles + p.dense - 1) / p.dense, p.min_tiles);
        p.dense = (tiles + p.dense_tiles - 1) / p.dense_tiles;
        p.items = B * p.dense;
        p.merge = p.dense > 1;
    }
    if (p.merge) {
        const size_t rows = (size_t)p.items * units * p.M;
        p.o_bytes = (rows * D * sizeof(_Float16) + 255) & ~(size_t)255;
        p.bytes = p.o_bytes + rows * sizeof(f32x4);
    }
    if (p.bytes < 256) p.bytes = 256;
    return p;
}

template <int MODE>
static int attn_run(const void* q, const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                    const int32_t* block_table, const int32_t* context_lens, const int32_t* vis, void* out, int B,
                    int Q, int Hq, int Hkv, int D_, int page_size, int block, int max_pages, int num_pages,
                    float scale, int max_context, void* workspace, size_t ws_bytes, void* stream) {
    if (B < 1 || B > 65535 || Q < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv) return D3D_E_SHAPE;
    if (D_ != D || Hq / Hkv > 64) return D3D_E_UNSUPPORTED;
    if (page_size < 1 || max_pages < 1 || num_pages < 1 || max_context < 1) return D3D_E_SHAPE;
    if ((int64_t)max_pages * page_size > INT_MAX / 2 || (int64_t)max_pages * page_size < max_context) return D3D_E_SHAPE;
    if ((int64_t)num_pages * page_size > INT_MAX / Hkv) return D3D_E_SHAPE;  // rows of a cache
    const int sh = fp8_block_shift(page_size, block);
    if (sh < 0) return D3D_E_UNSUPPORTED;
    if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !block_table || !context_lens || !out) return D3D_E_NULL;
    if (MODE == kPacked && !vis) return D3D_E_NULL;
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16)
        return D3D_E_UNSUPPORTED;
    const AttnPlan pl = attn_plan(B, Q, Hq, Hkv, max_context);
    if (pl.nqt > 65535 || (int64_t)B * pl.nqt > 65535 || (int64_t)pl.items * Hkv > INT_MAX / 512) return D3D_E_SHAPE;
    if (pl.merge && (!workspace || ws_bytes < pl.bytes || (uintptr_t)workspace % 16)) return D3D_E_WORKSPACE;
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
    P.part_o = static_cast<_Float16*>(workspace);
    P.part_ml = reinterpret_cast<f32x4*>(static_cast<char*>(workspace) + pl.o_bytes);
    P.B = B;
    P.Q = Q;
    P.Hq = Hq;
    P.Hkv = Hkv;
    P.G = Hq / Hkv;
    P.QT = pl.QT;
    P.nqt = pl.nqt;
    P.M = pl.M;
    P.page_size = page_size;
    P.block_shift = sh;
    P.max_pages = max_pages;
    P.num_pages = num_pages;
    P.max_context = max_context;
    P.items = pl.items;
    P.slots = pl.slots;
    P.min_tiles = pl.min_tiles;
    P.dense = pl.dense;
    P.dense_tiles = pl.dense_tiles;
    P.scale_log2 = scale * 1.4426950408889634f;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(pl.items * Hkv), (unsigned)pl.nqt);
    switch (pl.rt) {
        case 1: hipLaunchKernelGGL((attn_kernel<MODE, 1, 4>), grid, dim3(256), 0, s, P); break;
        case 2: hipLaunchKernelGGL((attn_kernel<MODE, 2, 4>), grid, dim3(256), 0, s, P); break;
        default: hipLaunchKernelGGL((attn_kernel<MODE, 4, 4>), grid, dim3(256), 0, s, P); break;
    }
    if (pl.merge)
        hipLaunchKernelGGL(attn_merge_kernel, dim3((unsigned)((P.M + kRows - 1) / kRows), (unsigned)Hkv, (unsigned)(B * pl.nqt)),
                           dim3(256), 0, s, P);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? D3D_OK : (int)err;
}

}  // namespace fp8
}  // namespace d3d

using namespace d3d;

extern "C" size_t d3d_attn_fp8_workspace_bytes(int B, int Q, int Hq, int Hkv, int D, int page_size, int max_context) {
    if (B < 1 || Q < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || D != fp8::D || page_size < 1 || max_context < 1 || Hq / Hkv > 64)
        return 0;
    return fp8::attn_plan(B, Q, Hq, Hkv, max_context).bytes;
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
