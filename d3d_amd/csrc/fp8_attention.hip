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
//
// What bounds it, with measured times (32 query and 8 KV heads): long contexts
// their bytes (two of 131,072 tokens, 16 queries: 102.3 us, 5.2 TB/s, the rate of
// a large copy; 48 single tokens over 192 MB: 41.9 us); prompts the issue of about
// 250 VALU (widening, exponentials, packing) beside 64 MFMA in a step of 64 rows (366
// GFLOP in 384 us); small calls the chain of dependent loads and the second
// launch (16 queries over 2,051 tokens: 9.0 + 4.0 us; one over 333: 7.3).
// Probabilities shared through LDS, the waves on their own output dimensions and a
// barrier per 128 tokens, measured slower (573 us against 481 for the prompts).
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
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

constexpr int NW = 4;           // waves of a workgroup
constexpr int kStep = 32;       // tokens a wave takes at a time
constexpr int kTile = 128;      // tokens four waves take at a time: the unit of ranges
// Tiles per range from which four row tiles take two workgroups per CU: a short
// range is mostly its own beginning and end, and more ranges mean more to merge
// (8 requests of 608 to 2,432 tokens and 16 rows: 17.0 + 5.0 us with one, 19.1
// + 5.5 with two; two of 131,072 tokens: 105 with one, 103 with two).
constexpr int kDeep = 16;
constexpr int kMaxTiles = 64;   // tiles of a range whose pages and scales are staged at once
constexpr int kVRow = D + 16;   // LDS bytes per value row: 16 rows, 36 banks apart, read without conflicts
constexpr float kNone = -3.0e38f;  // the reference of a row that has seen nothing: -inf without its special cases
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
    int qt_inv;      // 2^16 / QT rounded up: row / QT of rows below 64
    int page_shift;  // log2 of the page size, or -1
    int page_size, block_shift, max_pages, num_pages;
    int max_context;
    int items;   // ranges of all requests at most
    int room;      // ranges that run at once
    int room_one;  // the same with one workgroup per CU,
    int deep;      // where all contexts together have fewer tiles than this
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
    v += xor_desc<32>(v);
    v += xor_desc<16>(v);
    v += xor_desc<8>(v);
    v += xor_desc<4>(v);
    v += xor_desc<2>(v);
    return v + xor_desc<1>(v);
}

template <int O>
__device__ __forceinline__ int scan_step(int v, int lane) {
    const int t = (int)up_partner<O>((uint32_t)v);
    return lane >= O ? v + t : v;
}

__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// How the contexts are cut, the same in every workgroup of both launches.  Up
// to 64 requests: with about the least number of tiles per range that keeps
// the ranges of all requests within P.room workgroups; item numbers run through
// the requests' own range counts.  A whole wave calls it.
struct Range {
    int b, s, n, first;  // request (-1: none), range, ranges of the request, its first item
};

__device__ __forceinline__ int tiles_of(const AttnParams& P, int b) {
    return (max(ctx_of(P, b), 1) + kTile - 1) / kTile;
}

__device__ __forceinline__ int room_of(const AttnParams& P, int total) {
    return total >= P.deep ? P.room : P.room_one;
}

__device__ __forceinline__ void cut_of(const AttnParams& P, int lane, int& incl, int& n) {
    const int t = lane < P.B ? tiles_of(P, lane) : 0;
    const int total = wave_sum_int(t), room = room_of(P, total);
    // A request's last range is half full on average: aimed at fewer ranges by half
    // the requests the first try mostly fits (48 single tokens 43.4 + 5.3 us -> 41.9
    // + 4.7, packed block of 4 requests 35.0 + 6.6 -> 34.6 + 5.0).
    const int aim = max(1, room - P.B / 2);
    int tiles = max(P.min_tiles, (total + aim - 1) / aim);
    for (;;) {
        n = lane < P.B ? (t + tiles - 1) / tiles : 0;
        const int sum = wave_sum_int(n);
        if (sum <= max(room, P.B)) break;  // one range each at the least
        tiles += max(1, (int)((float)tiles * (float)(sum - room) / (float)(2 * sum)));
    }
    incl = scan_step<1>(n, lane);
    incl = scan_step<2>(incl, lane);
    incl = scan_step<4>(incl, lane);
    incl = scan_step<8>(incl, lane);
    incl = scan_step<16>(incl, lane);
    incl = scan_step<32>(incl, lane);
}

// One request: the same, without the wave.
__device__ __forceinline__ int cut_of_one(const AttnParams& P) {
    const int t = tiles_of(P, 0), room = room_of(P, t), tiles = max(P.min_tiles, (t + room - 1) / room);
    return (t + tiles - 1) / tiles;
}

__device__ __forceinline__ int cut_dense(const AttnParams& P, int b) {
    return (tiles_of(P, b) + P.dense_tiles - 1) / P.dense_tiles;
}

__device__ __forceinline__ Range range_of_item(const AttnParams& P, int item) {
    if (P.dense) {
        const int b = P.B - 1 - item / P.dense, s = item % P.dense;  // later requests first: a prompt's longer slices
        const int n = cut_dense(P, b);
        return {s < n ? b : -1, s, n, item - s};
    }
    if (P.B == 1) {
        const int n = cut_of_one(P);
        return {item < n ? 0 : -1, item, n, 0};
    }
    const int lane = threadIdx.x & 63;
    int incl, n;
    cut_of(P, lane, incl, n);
    const uint64_t past = __ballot(lane < P.B && incl > item);
    if (!past) return {-1, 0, 0, 0};
    const int b = __builtin_ctzll(past), nb = lane_value(n, b), first = lane_value(incl, b) - nb;
    return {b, item - first, nb, first};
}

__device__ __forceinline__ Range range_of_request(const AttnParams& P, int b) {
    if (P.dense) return {b, 0, cut_dense(P, b), (P.B - 1 - b) * P.dense};
    if (P.B == 1) return {0, 0, cut_of_one(P), 0};
    const int lane = threadIdx.x & 63;
    int incl, n;
    cut_of(P, lane, incl, n);
    const int nb = lane_value(n, b);
    return {b, 0, nb, lane_value(incl, b) - nb};
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

template <int MODE, int RT>
__global__ __launch_bounds__(NW * 64, 2) void attn_kernel(AttnParams P) {
    constexpr int NT = NW * 64, R = 16 * RT;
    constexpr int kGroups = kMaxTiles * kTile / 16;
    // Output exchange: half the dimensions at a time, a row's floats padded.
    constexpr int kHalf = D / 2, kORow = kHalf + 4;
    // Four row tiles' query operands stay in LDS: with them in registers too, one
    // wave fits a SIMD instead of two.
    constexpr bool QLDS = RT == 4;
    constexpr int kVBytes = NW * kStep * kVRow, kQBytes = QLDS ? RT * 4 * 64 * 16 : 0, kOBytes = NW * R * kORow * 4;
    __shared__ __attribute__((aligned(16))) char lds[kVBytes + kQBytes > kOBytes ? kVBytes + kQBytes : kOBytes];
    __shared__ int row_of[kGroups];      // first cache row of a 16-token group, -1: no page
    __shared__ u32x2 scale_of[kGroups];  // its key and value scales
    __shared__ float stat[2][NW][R];
    __shared__ int limit[MODE == kPacked ? 3 : 1][R];  // per row: visible keys t < [0], [1] <= t < [2]

    const int kvh = blockIdx.x % P.Hkv, qt = blockIdx.y, item = blockIdx.x / P.Hkv;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int g4 = lane >> 4, c16 = lane & 15;
    const Range rg = range_of_item(P, item);
    const int b = __builtin_amdgcn_readfirstlane(rg.b);
    if (b < 0) return;  // uniform, before any barrier
    const int n_ranges = __builtin_amdgcn_readfirstlane(rg.n);
    const int len = __builtin_amdgcn_readfirstlane(min(P.context_lens[b], P.max_pages * P.page_size));
    const int ctx = min(len, P.max_context), pre = len - P.Q, q0 = qt * P.QT;
    // The request's tiles in n_ranges even parts, the first ones a tile longer.
    const int tiles = (max(ctx, 1) + kTile - 1) / kTile, s_r = __builtin_amdgcn_readfirstlane(rg.s);
    const int part = tiles / n_ranges, longer = tiles - part * n_ranges;
    const int t_begin = (s_r * part + min(s_r, longer)) * kTile;
    const int t_last = min(t_begin + (part + (s_r < longer ? 1 : 0)) * kTile, ctx);

    // The page of a 16-token group of the piece from p0 on; -1 behind its end.
    const auto page_at = [&](int p0, int i) {
        const int t = p0 + 16 * i;
        if (i >= kGroups || t >= t_last) return -1;
        return P.block_table[(size_t)b * P.max_pages + (P.page_shift >= 0 ? t >> P.page_shift : t / P.page_size)];
    };
    int page = page_at(t_begin, threadIdx.x);  // on its way beside the queries

    // Q^T operands: dims 64 p + 16 g4 + 8 e .. + 7 at ks = 2 p + e, as the keys are
    // loaded.  Rows behind the last are a copy of row 0 that nobody writes out.
    const uint16_t* q_rows = P.q + ((size_t)b * P.Q * P.Hq + (size_t)kvh * P.G) * D + 16 * g4;
    const auto load_q = [&](int row, int ks) {
        const int gh = row * P.qt_inv >> 16, qi = q0 + row - gh * P.QT;
        const size_t at = row < P.M && qi < P.Q ? (size_t)qi * P.Hq + gh : 0;
        return *reinterpret_cast<const u32x4*>(q_rows + at * D + 64 * (ks >> 1) + 8 * (ks & 1));
    };
    bf16x8 qop[QLDS ? 1 : RT][4];
    if constexpr (QLDS) {
        static_assert(!QLDS || RT == NW, "a row tile per wave");
        u32x4 v[4];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) v[ks] = load_q(16 * w + c16, ks);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) *reinterpret_cast<u32x4*>(lds + kVBytes + ((w * 4 + ks) * 64 + lane) * 16) = v[ks];
    } else {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) qop[rt][ks] = __builtin_bit_cast(bf16x8, load_q(16 * rt + c16, ks));
    }

    // The rows' limits, a row per lane, kept in LDS: they are read where a step has
    // keys that some row does not see.  The frontier goes by the context's own
    // length, reads by its bounds.  Over all rows: keys below a_min are seen by
    // each, none from a_max on by any but [s_lo, s_hi).
    int a_min, a_max, s_lo = 0, s_hi = 0;
    {
        const int gh = lane * P.qt_inv >> 16, qi = q0 + lane - gh * P.QT;
        const bool row_ok = lane < P.M && qi < P.Q;
        int va = 0, lo = 0, hi = 0;
        if (row_ok) {
            va = ctx;
            if constexpr (MODE == kCausal) va = min(pre + qi + 1, ctx);
            if constexpr (MODE == kPacked) {
                va = min(pre + P.vis[qi * 3], ctx);
                lo = max(pre + P.vis[qi * 3 + 1], 0);
                hi = min(pre + P.vis[qi * 3 + 2], ctx);
            }
        }
        if (w == 0 && lane < R) {
            limit[0][lane] = va;
            if constexpr (MODE == kPacked) {
                limit[1][lane] = lo;
                limit[2][lane] = hi;
            }
        }
        if constexpr (MODE == kPacked) {
            const auto largest = [](int v) {
                v = max(v, xor_desc<32>(v));
                v = max(v, xor_desc<16>(v));
                v = max(v, xor_desc<8>(v));
                v = max(v, xor_desc<4>(v));
                v = max(v, xor_desc<2>(v));
                return __builtin_amdgcn_readfirstlane(max(v, xor_desc<1>(v)));
            };
            a_min = -largest(row_ok ? -va : -INT_MAX);
            a_max = largest(va);
            s_lo = -largest(lo < hi ? -lo : -INT_MAX);
            s_hi = largest(lo < hi ? hi : 0);
        } else if constexpr (MODE == kCausal) {
            a_min = min(pre + q0 + 1, ctx);
            a_max = min(pre + min(q0 + P.QT, P.Q), ctx);
        } else {
            a_min = a_max = ctx;
        }
    }

    f32x4 o[RT][8];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int n = 0; n < 8; ++n) o[rt][n] = {0.f, 0.f, 0.f, 0.f};
        m[rt] = kNone;
        l[rt] = 0.f;
    }

    bool first = true;  // nothing to rescale yet
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
        if (p0 != t_begin) page = page_at(p0, threadIdx.x);
        // A group's first row, and the place of its scales.
        const auto place = [&](int i, int pg, size_t& at) {
            int row = -1;
            at = 0;
            if (pg >= 0 && pg < P.num_pages) {
                const int t = p0 + 16 * i, in = P.page_shift >= 0 ? t & (P.page_size - 1) : t % P.page_size;
                const size_t ph = (size_t)pg * P.Hkv + kvh;
                at = ph * (P.page_size >> P.block_shift) + (in >> P.block_shift);
                row = (int)(ph * P.page_size + in);
            }
            row_of[i] = row;
            return row;
        };
        const auto put_scale = [&](int i, int row, size_t at) {
            scale_of[i] = row < 0 ? u32x2{0x3f800000u, 0x3f800000u}
                                  : u32x2{(uint32_t)P.k_scale[at] << 23, (uint32_t)P.v_scale[at] << 23};
        };
        size_t at;
        const int first_row = place(threadIdx.x, page, at);
        static_assert(kGroups == 2 * NT, "groups per thread");
        if (groups > NT) {  // uniform
            size_t at2;
            const int row2 = place(threadIdx.x + NT, page_at(p0, threadIdx.x + NT), at2);
            put_scale(threadIdx.x + NT, row2, at2);
        }
        __syncthreads();

        u32x4 kr[2][2], vr[4];
        const auto base_of = [&](int g) { return (size_t)max(__builtin_amdgcn_readfirstlane(row_of[g]), 0) * D; };
        const auto fetch_k = [&](int j) {
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const uint8_t* src = P.k_cache + base_of(2 * step_at(j) + sub);
#pragma unroll
                for (int p = 0; p < 2; ++p) kr[sub][p] = *reinterpret_cast<const u32x4*>(src + k_off + 64 * p);
            }
        };
        const auto fetch_v = [&](int j) {
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                const uint8_t* src = P.v_cache + base_of(2 * step_at(j) + sub);
#pragma unroll
                for (int p = 0; p < 2; ++p) vr[2 * sub + p] = *reinterpret_cast<const u32x4*>(src + v_off + 8 * D * p);
            }
        };
        if (w < steps) {
            fetch_k(w);
            fetch_v(w);
        }
        put_scale(threadIdx.x, first_row, at);  // beside the first keys and values
        __syncthreads();
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

            // sc[rt][sub][r]: token t0 + 16 sub + 4 g4 + r, row c16 of row tile rt.
            f32x4 sc[RT][2];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sc[rt][0] = sc[rt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    bf16x8 qf;
                    if constexpr (QLDS)
                        qf = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(lds + kVBytes + ((rt * 4 + ks) * 64 + lane) * 16));
                    else
                        qf = qop[rt][ks];
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub)
                        sc[rt][sub] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[sub][ks], qf, sc[rt][sub], 0, 0, 0);
                }
            // The next step's loads, behind the products that read the keys' registers.  Behind
            // the last step there is nothing to load, and a branch for it costs more than the
            // last step's again (batch-8 verify block 17.0 us instead of 16.3, prefill slices
            // 487 instead of 475: the products move behind it, and registers run out).
            fetch_k(min(j + NW, steps - 1));
            fetch_v(min(j + NW, steps - 1));
            if (edge) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const int row = 16 * rt + c16, va = min(limit[0][row], p_end);
                    const int lo = MODE == kPacked ? limit[MODE == kPacked ? 1 : 0][row] : 0;
                    const int hi = MODE == kPacked ? min(limit[MODE == kPacked ? 2 : 0][row], p_end) : 0;
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub) {
                        const int t = t0 + 16 * sub + 4 * g4;
                        f32x4 x = sc[rt][sub];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int hide = (int)(t + r >= va) & ((int)(t + r < lo) | (int)(t + r >= hi));
                            x[r] = hide ? -INFINITY : x[r];
                        }
                        sc[rt][sub] = x;
                    }
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
                    if (!first) {
                        const float alpha = __builtin_amdgcn_exp2f(m[rt] - mn);
                        l[rt] *= alpha;
#pragma unroll
                        for (int n = 0; n < 8; ++n) o[rt][n] *= alpha;
                    }
                    m[rt] = mn;
                }
            }
            first = false;
            // Probabilities as bf16 add 2^-9 of each; over many rows that is less than the
            // results' own rounding.  A few rows (single tokens) may put all weight on two
            // or three keys, where it showed (2.5 times the error of the result's rounding):
            // there a second bf16 holds what the first leaves.  The products hide under the
            // reads of a full card (48 requests of one token 43.6 us with either; one of
            // 333 tokens 7.0 -> 7.5).
            constexpr bool kTwo = RT == 1;
            bf16x8 pop[RT], rest[kTwo ? RT : 1];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                uint32_t pw[4], pr[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[rt][i >> 1][2 * (i & 1)], P.scale_log2, -m[rt]));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[rt][i >> 1][2 * (i & 1) + 1], P.scale_log2, -m[rt]));
                    pw[i] = pack_bf16x2(p0, p1);
                    if constexpr (kTwo) {
                        pr[i] = pack_bf16x2(p0 - __uint_as_float(pw[i] << 16), p1 - __uint_as_float(pw[i] & 0xffff0000u));
                        l[rt] += p0 + p1;
                    } else {
                        // The sum takes the rounded probabilities, as the product does.
                        l[rt] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pw[i]), bf16x2{(__bf16)1.f, (__bf16)1.f}, l[rt], false);
                    }
                }
                if constexpr (kTwo) rest[rt] = __builtin_bit_cast(bf16x8, u32x4{pr[0], pr[1], pr[2], pr[3]});
                pop[rt] = __builtin_bit_cast(bf16x8, u32x4{pw[0], pw[1], pw[2], pw[3]});
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const u32x2 c = lds_read_tr8(vbuf + (8 * g4 + (c16 >> 1)) * kVRow + 16 * n + 8 * (c16 & 1));
                const bf16x8 vf = widen8(c[0], c[1], vs0, vs1);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    o[rt][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pop[rt], o[rt][n], 0, 0, 0);
                    if constexpr (kTwo) o[rt][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, rest[rt], o[rt][n], 0, 0, 0);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (poison) {
                // Rows that see a NaN value: its dimension is NaN.
                for (int tok = 0; tok < kStep; ++tok) {
                    const int t = t0 + tok, at = row_of[g + (tok >> 4)];
                    if (t >= p_end || at < 0) continue;
                    const uint32_t* src = reinterpret_cast<const uint32_t*>(P.v_cache + ((size_t)at + (tok & 15)) * D) + g4;
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const uint32_t nb = nan_bytes(src[4 * n]);
                        if (!nb) continue;
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            const int row = 16 * rt + c16;
                            int see = (int)(t < limit[0][row]);
                            if constexpr (MODE == kPacked) see |= (int)(t >= limit[1][row]) & (int)(t < limit[2][row]);
                            f32x4 x = o[rt][n];
#pragma unroll
                            for (int r = 0; r < 4; ++r) x[r] = (see & (int)(nb >> (8 * r))) & 1 ? NAN : x[r];
                            o[rt][n] = x;
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
    // Thread tid adds up dims dp .. of row tr; TPR threads per row.
    constexpr int TPR = NT / R, DPT = kHalf / TPR;
    static_assert(TPR >= 1 && TPR <= 64 && DPT >= 1, "threads per row");
    const int tr = threadIdx.x / TPR, dp = (threadIdx.x % TPR) * DPT;
    float rm = kNone, rl = 0.f, fv[NW];
#pragma unroll
    for (int v = 0; v < NW; ++v) rm = fmaxf(rm, stat[0][v][tr]);
#pragma unroll
    for (int v = 0; v < NW; ++v) {
        fv[v] = __builtin_amdgcn_exp2f(stat[0][v][tr] - rm);
        rl = __builtin_fmaf(fv[v], stat[1][v][tr], rl);
    }
    const float inv = rl == 0.f ? 0.f : 1.f / rl;
#pragma unroll
    for (int v = 0; v < NW; ++v) fv[v] *= inv;
    const int orow_h = tr * P.qt_inv >> 16, orow_q = q0 + tr - orow_h * P.QT;
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
                *reinterpret_cast<f32x4*>(ex + (w * R + 16 * rt + c16) * kORow + 16 * n + 4 * g4) = o[rt][4 * half + n];
        __syncthreads();
        float sum[DPT];
#pragma unroll
        for (int d = 0; d < DPT; ++d) {
            sum[d] = 0.f;
#pragma unroll
            for (int v = 0; v < NW; ++v) sum[d] = __builtin_fmaf(fv[v], ex[(v * R + tr) * kORow + dp + d], sum[d]);
        }
        if (n_ranges == 1) {
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
            if constexpr (TPR >= 2) amax = fmaxf(amax, xor_asc<1>(amax));
            if constexpr (TPR >= 4) amax = fmaxf(amax, xor_asc<2>(amax));
            if constexpr (TPR >= 8) amax = fmaxf(amax, xor_asc<4>(amax));
            if constexpr (TPR >= 16) amax = fmaxf(amax, xor_asc<8>(amax));
            static_assert(TPR <= 16, "lanes of a row");
            const int e = min(max((int)((__float_as_uint(amax) >> 23) & 0xffu) - 127 - 14, -110), 110);
            es[half] = pow2(e);
            if (tr < P.M) {
                _Float16* dst = P.part_o + (unit * P.M + tr) * D + kHalf * half + dp;
#pragma unroll
                for (int d = 0; d < DPT; ++d) dst[d] = (_Float16)(sum[d] * pow2(-e));
            }
        }
    }
    if (n_ranges > 1 && tr < P.M && threadIdx.x % TPR == 0) P.part_ml[unit * P.M + tr] = f32x4{rm, rl, es[0], es[1]};
}

// Merges the ranges of a request.  Sixteen lanes of 8 dims take every GR-th range
// of a row, four of them at once: a wave per row (GR = 4) where a request has
// many ranges, four rows per wave (GR = 1) where it has few.
template <int GR>
__global__ __launch_bounds__(256) void attn_merge_kernel(AttnParams P) {
    const int b = blockIdx.z / P.nqt, qt = blockIdx.z - b * P.nqt, kvh = blockIdx.y;
    const int lane = threadIdx.x & 63, grp = GR == 4 ? lane >> 4 : 0, d8 = (lane & 15) * 8;
    const int row = GR == 4 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x * 16 + (threadIdx.x >> 4);
    const Range rg = range_of_request(P, b);
    const int n = __builtin_amdgcn_readfirstlane(rg.n);
    if (n == 1) return;  // written by the first launch
    const int gh = row * P.qt_inv >> 16, q = qt * P.QT + row - gh * P.QT;
    const bool live = row < P.M && q < P.Q;
    const size_t u0 = (((size_t)__builtin_amdgcn_readfirstlane(rg.first) * P.nqt + qt) * P.Hkv + kvh) * P.M + (live ? row : 0);
    const size_t du = (size_t)P.nqt * P.Hkv * P.M;
    float m = kNone, den = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s0 = grp; s0 < n; s0 += 4 * GR) {
        f32x4 ml[4];
        h16x8 o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const size_t u = u0 + (size_t)min(s0 + GR * k, n - 1) * du;
            ml[k] = P.part_ml[u];
            o[k] = *reinterpret_cast<const h16x8*>(P.part_o + u * D + d8);
        }
        float mn = m;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (s0 + GR * k >= n) ml[k] = f32x4{kNone, 0.f, 0.f, 0.f};  // the last range's again: not twice
            mn = fmaxf(mn, ml[k][0]);
        }
        const float keep = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        den *= keep;
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[d] *= keep;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float wgt = __builtin_amdgcn_exp2f(ml[k][0] - mn) * ml[k][1];
            den += wgt;
            const float f = wgt * (d8 < 64 ? ml[k][2] : ml[k][3]);
            if (s0 + GR * k < n) {  // a NaN that was counted already times 0
#pragma unroll
                for (int d = 0; d < 8; ++d) acc[d] = __builtin_fmaf(f, (float)o[k][d], acc[d]);
            }
        }
    }
    if constexpr (GR == 4) {
        const float f = __builtin_amdgcn_exp2f(m - across_max(m));
        den = across_sum(den * f);
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[d] = across_sum(acc[d] * f);
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    if (live && grp == 0)
        *reinterpret_cast<u32x4*>(P.out + (((size_t)b * P.Q + q) * P.Hq + kvh * P.G + gh) * D + d8) =
            u32x4{pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                  pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv)};
}

constexpr int kMaxRanges = 512;  // of a request

struct AttnPlan {
    int QT, nqt, M, rt, items, room, room_one, deep, min_tiles, dense, dense_tiles;
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
    // Workgroups that run at once: three per CU with one row tile, two with more.
    const int64_t units = (int64_t)Hkv * p.nqt;
    const auto room = [&](int slots) { return (int)std::max<int64_t>(slots / units, 1); };
    p.room = room(p.rt == 1 ? 768 : 512);
    p.room_one = p.rt == 4 ? room(256) : p.room;
    p.deep = kDeep * p.room_one;
    p.min_tiles = p.rt == 1 ? 4 : 1;
    const int tiles = (max_context + kTile - 1) / kTile;
    if (B <= 64) {
        p.items = std::max(B, p.room);
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
    if (!(scale > 0.f && scale < INFINITY)) return D3D_E_UNSUPPORTED;  // a masked score is -inf times it
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
    P.qt_inv = (65536 + pl.QT - 1) / pl.QT;
    P.page_shift = -1;
    if ((page_size & (page_size - 1)) == 0) P.page_shift = __builtin_ctz((unsigned)page_size);
    P.page_size = page_size;
    P.block_shift = sh;
    P.max_pages = max_pages;
    P.num_pages = num_pages;
    P.max_context = max_context;
    P.items = pl.items;
    P.room = pl.room;
    P.room_one = pl.room_one;
    P.deep = pl.deep;
    P.min_tiles = pl.min_tiles;
    P.dense = pl.dense;
    P.dense_tiles = pl.dense_tiles;
    P.scale_log2 = scale * 1.4426950408889634f;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(pl.items * Hkv), (unsigned)pl.nqt);
    switch (pl.rt) {
        case 1: hipLaunchKernelGGL((attn_kernel<MODE, 1>), grid, dim3(256), 0, s, P); break;
        case 2: hipLaunchKernelGGL((attn_kernel<MODE, 2>), grid, dim3(256), 0, s, P); break;
        default: hipLaunchKernelGGL((attn_kernel<MODE, 4>), grid, dim3(256), 0, s, P); break;
    }
    if (pl.merge) {
        const unsigned y = (unsigned)Hkv, z = (unsigned)(B * pl.nqt);
        if (pl.items > 4 * B)
            hipLaunchKernelGGL((attn_merge_kernel<4>), dim3((unsigned)((P.M + 3) / 4), y, z), dim3(256), 0, s, P);
        else
            hipLaunchKernelGGL((attn_merge_kernel<1>), dim3((unsigned)((P.M + 15) / 16), y, z), dim3(256), 0, s, P);
    }
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? D3D_OK : (int)err;
}

}  // namespace fp8
}  // namespace d3d

using namespace d3d;

extern "C" size_t d3d_attn_fp8_workspace_bytes(int B, int Q, int Hq, int Hkv, int D, int page_size, int max_context) {
    if (B < 1 || Q < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || D != fp8::D || page_size < 1 || max_context < 1 ||
        max_context > INT_MAX / 2 || Hq / Hkv > 64)
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
