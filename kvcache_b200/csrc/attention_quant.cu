// Attention of few query rows over cache pages in eight bits (csrc/cache_quant.cuh): single tokens and short portions, bfloat16
// queries and results, compiled per head size with -DKVB_HEAD_DIM=32, 64, 96 or 128.
//
// It computes what the reference's k_batched_paged_decode_attn computes (src/qwen_kernels.cu:293-335), split over keys and merged as
// src/flash_decode.cu:82-101 does, from codes c and exponents e instead of half-precision rows:
//   score_j = scale 2^(e_j) (q . c_j),   out = sum_j w_j 2^(f_j) d_j / sum_j w_j,   w_j = 2^(score_j log2 e)
// with (c, e) a key's and (d, f) a value's row.  The weights that meet the value codes are n_j = 2^(score_j log2 e + f_j - m), m the
// largest of those exponents so far: at most 1, and what matters for the sum is near 1 whatever the rows' scales are, so that half
// precision holds them to 2^-11.  The denominator takes n_j 2^(-f_j), in float32.  Codes are exact in half precision, and so
// are queries once a power of two has brought their row to about 1: products run on mma.sync m16n8k16 (half, float32 sums),
// whose 16 rows are the query heads that share a key head (times the tokens of a short portion).
//
// A warp takes 32 keys at a time and needs nothing from any other until its run ends.  The order of an MMA's inner index is free as
// long as both operands agree, so a lane's share of a tile is bytes that lie together: for the scores 16 (or 8) of a key's
// numbers, for the sum the same of four neighbouring keys' values.  Each lane copies those bytes itself (cp.async, into slots of
// shared memory that no other lane touches), several tiles ahead, and turns them into half precision in registers: no barrier, no
// bank conflict and no wait for another lane stands in the stream.
//
// Work is shared out by keys: units of 128 keys of every (segment, key head, tile of 16 rows), laid end to end, are cut into equal
// runs, one a block, whatever the lengths.  Where a cut divides a row tile's keys, the pieces' sums meet in scratch, two places a
// block, and the last piece to finish adds them in order (a ticket per block): the same bits whichever is last.
#include "cache_quant.cuh"
#include <type_traits>

#ifndef KVB_HEAD_DIM
#error "compile with -DKVB_HEAD_DIM=32, 64, 96 or 128"
#endif

namespace aq {
using namespace cq;

constexpr int D = KVB_HEAD_DIM;
static_assert(D == 32 || D == 64 || D == 96 || D == 128, "head sizes 32, 64, 96 and 128");
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int WARP_KEYS = 32, UNIT = WARPS * WARP_KEYS;
constexpr int KU = D % 64 == 0 ? 16 : 8, KN = D / (4 * KU);                       // bytes a copy, copies a key row and lane: four lanes share a key row
constexpr int VU = D % 128 == 0 ? 16 : D % 64 == 0 ? 8 : 4, VN = D / (8 * VU);    // ... eight lanes share a value row
constexpr int K_BYTES = 4 * KN * KU * 32, V_BYTES = 8 * VN * VU * 32, STAGE_BYTES = K_BYTES + V_BYTES + 4 * 32 * 4;
constexpr int STAGES = D == 128 ? 3 : 4;
constexpr int WARP_BYTES = STAGES * STAGE_BYTES;
constexpr int O_STRIDE = D + 4;
constexpr int BLOCKS_PER_SM = D == 128 ? 2 : D == 96 ? 2 : 3;
static_assert(16 * O_STRIDE * 4 + 128 <= WARP_BYTES, "a warp's sums lie over its slots");
constexpr int MAX_SEGMENTS = 4096;
constexpr int PIECE_COST = 1;          // what a piece costs beside its keys, in units
constexpr float NEG_INF = -INFINITY;

struct Params {
    const bf16* q;             // [T, Hq * D]
    bf16* out;
    const uint8_t* k_codes;    // [num_pages, Hkv, page_size, D]
    const uint8_t* v_codes;
    const uint8_t* k_scales;   // [num_pages, Hkv, page_size]
    const uint8_t* v_scales;
    int num_pages;
    const int* block_table;
    int table_stride, page_shift;
    int segments;
    const int* seg_q_start;
    const int* seg_q_len;
    const int* seg_kv_len;
    int max_q;                 // segments of more tokens are left out
    int Hq, Hkv, group, reach, keep;
    float scale, cap;
    const float* sink;
    const float* slopes;
    float* part_o;             // [2 * blocks, 16, D]
    float* part_ml;            // [2 * blocks, 16, 2]
    int* tickets;              // [blocks], zero between launches
    int min_units;
    int* err;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool there) {
    const int n = there ? BYTES : 0;                       // the rest is filled with zeros
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(from), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(to), "l"(from), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
template <int BYTES> __device__ __forceinline__ void read_slot(uint32_t from, uint32_t* w) {
    if (BYTES == 16) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(from) : "memory");
    else if (BYTES == 8) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(w[0]), "=r"(w[1]) : "r"(from) : "memory");
    else asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(w[0]) : "r"(from) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// c += a b; rows 8 to 15 of a are zero where HALF_ROWS.
template <bool HALF_ROWS>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(HALF_ROWS ? 0u : a[1]), "r"(a[HALF_ROWS ? 1 : 2]), "r"(HALF_ROWS ? 0u : a[3]), "r"(b0), "r"(b1));
}
// Two neighbouring codes of a word (the lower or the upper two bytes) as half precision.  int8: the bytes, with their sign bits
// flipped (`flipped`), become the low bits of 1024 + c + 128, from which 1152 is taken.
template <int STORE> __device__ __forceinline__ uint32_t flipped(uint32_t w) { return STORE == KVB_INT8 ? w ^ 0x80808080u : w; }
template <int STORE, int UPPER>
__device__ __forceinline__ uint32_t halves(uint32_t w) {
    if (STORE == KVB_INT8) {
        const uint32_t v = __byte_perm(w, 0x64646464u, UPPER ? 0x4342 : 0x4140);
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&v), __half2half2(__ushort_as_half(0x6480)));
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(UPPER ? w >> 16 : w & 0xffffu), __NV_E4M3);
    return (uint32_t)h.x | ((uint32_t)h.y << 16);
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A segment's line of units, and one of its row tiles.
struct Segment {
    int q_start, q_len, start, keep;
    int tile_begin, n_keep, n;         // the list of units: n_keep units of kept keys, then from unit tile_begin on
    int row_tiles;
};
__device__ __forceinline__ Segment make_segment(const Params& p, int s) {
    Segment c;
    c.q_start = p.seg_q_start[s];
    c.q_len = p.seg_q_len[s];
    const int kv_len = p.seg_kv_len[s];
    if (c.q_len > p.max_q || c.q_len < 1 || kv_len < c.q_len) { c.q_len = c.row_tiles = c.n = 0; return c; }
    c.start = kv_len - c.q_len;
    c.keep = p.reach > 0 ? p.keep : 0;
    c.tile_begin = first_seen_key(c.start, p.reach) / UNIT;
    c.n_keep = min((c.keep + UNIT - 1) / UNIT, c.tile_begin);
    c.n = c.n_keep + (kv_len - 1) / UNIT + 1 - c.tile_begin;
    c.row_tiles = (c.q_len * p.group + 15) >> 4;
    return c;
}

template <int STORE, bool HALF_ROWS>
__global__ void __launch_bounds__(THREADS, BLOCKS_PER_SM) attention_quant_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int RG = HALF_ROWS ? 1 : 2;                   // rows a lane has: g, and g + 8
    int* const first = reinterpret_cast<int*>(smem + WARPS * WARP_BYTES);     // [segments + 1] the line before each segment
    __shared__ int scan_s[WARPS + 1], ticket_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

    // The step's lengths are metadata that no kernel before this one writes.
    int before = 0;
    for (int base = 0; base < p.segments; base += THREADS) {
        int mine = 0;
        if (base + tid < p.segments) { const Segment c = make_segment(p, base + tid); mine = c.row_tiles * p.Hkv * (c.n + PIECE_COST); }
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += up; }
        if (lane == 31) scan_s[warp] = sum;
        __syncthreads();
        int below = before, all = before;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) { if (w < warp) below += scan_s[w]; all += scan_s[w]; }
        if (base + tid < p.segments) first[base + tid] = below + sum - mine;
        before = all;
        __syncthreads();
    }
    if (tid == 0) first[p.segments] = before;
    __syncthreads();
    const int total = before;
    const int share = max(p.min_units, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    const int w_begin = (int)min((long long)total, (long long)blockIdx.x * share), w_end = min(total, w_begin + share);
    int seg = 0;
    for (int hi = p.segments; hi - seg > 1;) { const int mid = (seg + hi) >> 1; if (first[mid] <= w_begin) seg = mid; else hi = mid; }
    pdl_wait();
    pdl_launch_dependents();

    unsigned char* const mine = smem + warp * WARP_BYTES;
    const uint32_t slots = smem_addr(mine);
    const int page_mask = (1 << p.page_shift) - 1;

    for (int w = w_begin; w < w_end;) {
        while (first[seg + 1] <= w) ++seg;
        const Segment c = make_segment(p, seg);
        const int per = c.n + PIECE_COST, off = w - first[seg], item = off / per, at = off - item * per;
        const int to = min(per, at + w_end - w);
        const int item_first = w - at + PIECE_COST;          // where the row tile's first unit lies in the line
        const int begin = max(0, at - PIECE_COST), end = max(begin, to - PIECE_COST);
        w += to - at;
        if (begin == end) continue;
        const int hk = item / c.row_tiles, row0 = (item - hk * c.row_tiles) << 4;
        const int rows = min(16, c.q_len * p.group - row0);
        const int pos_first = c.start + row0 / p.group, pos_last = c.start + (row0 + rows - 1) / p.group;
        const int lo_first = first_seen_key(pos_first, p.reach), lo_last = first_seen_key(pos_last, p.reach);
        const int* const table = p.block_table + (size_t)seg * p.table_stride;

        // This lane's rows: queries as fragments, brought to about 1 by a power of two that goes into the score's factor.
        uint32_t qf[KN * KU / 4][2 * RG];
        float factor[RG], slope[RG];
        int pos[RG], lo[RG];
#pragma unroll
        for (int r = 0; r < RG; ++r) {
            const int row = row0 + g + 8 * r, token = row / p.group, head = hk * p.group + row - token * p.group;
            const bool there = g + 8 * r < rows;
            pos[r] = there ? c.start + token : 0;
            lo[r] = first_seen_key(pos[r], p.reach);
            slope[r] = there && p.slopes ? p.slopes[head] : 0.f;
            uint2 raw[KN * KU / 4];
            uint32_t top = 0u;
            const bf16* const from = p.q + ((size_t)(c.q_start + token) * p.Hq + head) * D + t * KU;
#pragma unroll
            for (int k = 0; k < KN * KU / 4; ++k) {
                raw[k] = there ? *reinterpret_cast<const uint2*>(from + (k / (KU / 4)) * 4 * KU + (k % (KU / 4)) * 4) : make_uint2(0u, 0u);
                top = max(top, max(max(raw[k].x & 0x7fffu, (raw[k].x >> 16) & 0x7fffu), max(raw[k].y & 0x7fffu, (raw[k].y >> 16) & 0x7fffu)));
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = top == 0u || top >= 0x7f80u ? 0 : min(100, max(-100, (int)(top >> 7) - 127));
            const float down = __int_as_float((127 - e) << 23);
            factor[r] = p.scale * __int_as_float((127 + e) << 23);
#pragma unroll
            for (int k = 0; k < KN * KU / 4; ++k) {
                qf[k][r] = pack(__uint_as_float(raw[k].x << 16) * down, __uint_as_float(raw[k].x & 0xffff0000u) * down);
                qf[k][RG + r] = pack(__uint_as_float(raw[k].y << 16) * down, __uint_as_float(raw[k].y & 0xffff0000u) * down);
            }
        }
        const bool biased = p.cap > 0.f || p.slopes;
        if (!biased)
#pragma unroll
            for (int r = 0; r < RG; ++r) factor[r] *= 1.4426950408889634f;

        auto key_of = [&](int i) -> int { return (i < c.n_keep ? i : c.tile_begin - c.n_keep + i) * UNIT + warp * WARP_KEYS; };
        // Pages of the four neighbouring keys that hold this lane's key rows and value rows, of both halves of 32 keys.
        int page_k[2], page_v[2];
        auto page_of = [&](int key) -> int {
            if (key > pos_last || (key + 3 < lo_first && key >= c.keep)) return -1;
            const int place = key >> p.page_shift;
            const int page = place < p.table_stride ? __ldg(table + place) : -1;
            if (page >= 0 && page < p.num_pages) return page;
            atomicOr(p.err, KVB_DEV_BAD_PAGE);
            return -1;
        };
        auto lookup = [&](int i) {
            if (i >= end) return;
            const int key0 = key_of(i);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                page_k[s] = page_of(key0 + 16 * s + 4 * (g >> 1));
                page_v[s] = page_of(key0 + 16 * s + 4 * t);
            }
        };
        auto fetch = [&](int i, int stage) {
            if (i < end) {
                const int key0 = key_of(i);
                const uint32_t base = slots + stage * STAGE_BYTES;
                auto seen = [&](int key) { return key <= pos_last && (key >= lo_first || key < c.keep); };
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int kk = key0 + 16 * s + 4 * (g >> 1), vv = key0 + 16 * s + 4 * t;
                    const bool has_k = page_k[s] >= 0, has_v = page_v[s] >= 0;
                    const size_t row_k = has_k ? ((((size_t)page_k[s] * p.Hkv + hk) << p.page_shift) + (kk & page_mask)) : 0;
                    const size_t row_v = has_v ? ((((size_t)page_v[s] * p.Hkv + hk) << p.page_shift) + (vv & page_mask)) : 0;
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const int more = 2 * n + (g & 1);
                        const bool there = has_k && seen(kk + more);
                        const uint8_t* const from = p.k_codes + (there ? (row_k + more) * D + t * KU : 0);
#pragma unroll
                        for (int u = 0; u < KN; ++u)
                            copy_async<KU>(base + (((s * 2 + n) * KN + u) * 32 + lane) * KU, from + u * 4 * KU, there);
                    }
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) {
                        const bool there = has_v && seen(vv + i4);
                        const uint8_t* const from = p.v_codes + (there ? (row_v + i4) * D + g * VU : 0);
#pragma unroll
                        for (int u = 0; u < VN; ++u)
                            copy_async<VU>(base + K_BYTES + (((s * 4 + i4) * VN + u) * 32 + lane) * VU, from + u * 8 * VU, there);
                    }
                    copy_async<4>(base + K_BYTES + V_BYTES + (2 * s * 32 + lane) * 4, p.k_scales + row_v, has_v);
                    copy_async<4>(base + K_BYTES + V_BYTES + ((2 * s + 1) * 32 + lane) * 4, p.v_scales + row_v, has_v);
                }
            }
            copies_commit();
        };

        float o[VN * VU][4];
#pragma unroll
        for (int i = 0; i < VN * VU; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m[RG], l[RG];
#pragma unroll
        for (int r = 0; r < RG; ++r) { m[r] = NEG_INF; l[r] = 0.f; }

        // 32 keys from `key0` on, whose bytes are there.  MASKED: some row may miss one of them.
        auto tile = [&](int key0, int stage, auto masked_tag) {
            constexpr bool MASKED = decltype(masked_tag)::value;
            const uint32_t base = slots + stage * STAGE_BYTES;
            float s[2][2][4];
            uint32_t kb[2], vb[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int n = 0; n < 2; ++n) s[h][n][0] = s[h][n][1] = s[h][n][2] = s[h][n][3] = 0.f;
                read_slot<4>(base + K_BYTES + V_BYTES + (2 * h * 32 + lane) * 4, &kb[h]);
                read_slot<4>(base + K_BYTES + V_BYTES + ((2 * h + 1) * 32 + lane) * 4, &vb[h]);
#pragma unroll
                for (int u = 0; u < KN; ++u)
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        uint32_t word[KU / 4];
                        read_slot<KU>(base + (((h * 2 + n) * KN + u) * 32 + lane) * KU, word);
#pragma unroll
                        for (int k = 0; k < KU / 4; ++k) {
                            const uint32_t x = flipped<STORE>(word[k]);
                            mma<HALF_ROWS>(s[h][n], qf[u * (KU / 4) + k], halves<STORE, 0>(x), halves<STORE, 1>(x));
                        }
                    }
            }
            // Exponents of the weights that the value codes get: score (base 2) + the value row's exponent.
            float top[RG], inv[2][4];
#pragma unroll
            for (int r = 0; r < RG; ++r) top[r] = NEG_INF;
            uint32_t hidden[RG];
#pragma unroll
            for (int r = 0; r < RG; ++r) hidden[r] = 0u;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int kbyte = (kb[h] >> (8 * i)) & 255, vbyte = (vb[h] >> (8 * i)) & 255;
                    const float up = __int_as_float(kbyte << 23);
                    const float shift = __int_as_float(0x4b000000 | vbyte) - 8388735.f;           // vbyte - 127
                    inv[h][i] = __int_as_float((254 - vbyte) << 23);                              // -infinity for a row that is not finite
                    const int key = key0 + 16 * h + 4 * t + i;
#pragma unroll
                    for (int r = 0; r < RG; ++r) {
                        float x = s[h][i >> 1][(i & 1) + 2 * r] * up * factor[r];
                        if (biased) {
                            if (p.cap > 0.f) x = p.cap * (1.f - __fdividef(2.f, 1.f + ex2(x / p.cap * 2.885390081777927f)));
                            x = (x - slope[r] * (float)(pos[r] - key)) * 1.4426950408889634f;
                        }
                        x += shift;
                        if (MASKED && !(key <= pos[r] && (key >= lo[r] || key < c.keep))) { x = NEG_INF; hidden[r] |= 1u << (4 * h + i); }
                        s[h][i >> 1][(i & 1) + 2 * r] = x;
                        top[r] = fmaxf(top[r], x);
                    }
                }
            bool moved = false;
            float base_m[RG], corr[RG];
#pragma unroll
            for (int r = 0; r < RG; ++r) {
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                const float now = fmaxf(m[r], top[r]);
                base_m[r] = now == NEG_INF ? 0.f : now;
                corr[r] = ex2(m[r] - base_m[r]);
                moved |= now > m[r];
                m[r] = now;
                l[r] *= corr[r];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < RG; ++r) {
                        float& x = s[h][i >> 1][(i & 1) + 2 * r];
                        x = ex2(x - base_m[r]);
                        l[r] = fmaf(x, MASKED && ((hidden[r] >> (4 * h + i)) & 1u) ? 0.f : inv[h][i], l[r]);
                    }
            if (__any_sync(0xffffffffu, moved)) {            // the maxima seldom move once a few tiles are in
#pragma unroll
                for (int i = 0; i < VN * VU; ++i)
#pragma unroll
                    for (int e = 0; e < 2 * RG; ++e) o[i][e] *= corr[e >> 1];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t pa[2 * RG];
#pragma unroll
                for (int r = 0; r < RG; ++r) {
                    pa[r] = pack(s[h][0][2 * r], s[h][0][2 * r + 1]);
                    pa[RG + r] = pack(s[h][1][2 * r], s[h][1][2 * r + 1]);
                }
#pragma unroll
                for (int u = 0; u < VN; ++u) {
                    uint32_t v[4][VU / 4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) read_slot<VU>(base + K_BYTES + (((h * 4 + i) * VN + u) * 32 + lane) * VU, v[i]);
#pragma unroll
                    for (int k = 0; k < VU / 4; ++k) {
                        // Four keys' words, a byte a column: bytes of neighbouring keys side by side.
                        const uint32_t a_lo = flipped<STORE>(__byte_perm(v[0][k], v[1][k], 0x5140)), a_hi = flipped<STORE>(__byte_perm(v[0][k], v[1][k], 0x7362));
                        const uint32_t b_lo = flipped<STORE>(__byte_perm(v[2][k], v[3][k], 0x5140)), b_hi = flipped<STORE>(__byte_perm(v[2][k], v[3][k], 0x7362));
                        float(*const to)[4] = &o[u * VU + 4 * k];
                        mma<HALF_ROWS>(to[0], pa, halves<STORE, 0>(a_lo), halves<STORE, 0>(b_lo));
                        mma<HALF_ROWS>(to[1], pa, halves<STORE, 1>(a_lo), halves<STORE, 1>(b_lo));
                        mma<HALF_ROWS>(to[2], pa, halves<STORE, 0>(a_hi), halves<STORE, 0>(b_hi));
                        mma<HALF_ROWS>(to[3], pa, halves<STORE, 1>(a_hi), halves<STORE, 1>(b_hi));
                    }
                }
            }
        };

        lookup(begin);
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) { fetch(begin + s, s); lookup(begin + s + 1); }
        int stage = 0;
        for (int i = begin; i < end; ++i) {
            // The slots that the next fetch fills were read by this lane alone, in the turn before.
            const int key0 = key_of(i);
            fetch(i + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
            lookup(i + STAGES);
            copies_wait<STAGES - 1>();
            if (key0 <= pos_last && (key0 + WARP_KEYS > lo_first || key0 < c.keep)) {
                if (key0 + WARP_KEYS - 1 <= pos_first && key0 >= lo_last) tile(key0, stage, std::false_type{});
                else tile(key0, stage, std::true_type{});
            }
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        copies_wait<0>();

        // The warps' sums meet in shared memory, over the slots.
        __syncwarp();
        float* const o_s = reinterpret_cast<float*>(mine);
        float* const ml_s = o_s + 16 * O_STRIDE;
#pragma unroll
        for (int r = 0; r < RG; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
#pragma unroll
            for (int u = 0; u < VN; ++u)
#pragma unroll
                for (int b = 0; b < VU; b += 4)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float(*const x)[4] = &o[u * VU + b];
                        *reinterpret_cast<float4*>(o_s + (g + 8 * r) * O_STRIDE + 8 * VU * u + VU * (2 * t + e) + b) =
                            make_float4(x[0][2 * r + e], x[1][2 * r + e], x[2][2 * r + e], x[3][2 * r + e]);
                    }
            if (t == 0) { ml_s[2 * (g + 8 * r)] = m[r]; ml_s[2 * (g + 8 * r) + 1] = l[r]; }
        }
        __syncthreads();
        const int block0 = item_first / share, block1 = (item_first + c.n - 1) / share;
        auto place_of = [&](int b) -> size_t { return (size_t)2 * b + (b * share > item_first ? 0 : 1); };
        auto store_row = [&](int r, int col, float4 x, float M, float L) {
            const int row = row0 + r, token = row / p.group, head = hk * p.group + row - token * p.group;
            if (p.sink) L += ex2(p.sink[head] * 1.4426950408889634f - (M == NEG_INF ? 0.f : M));
            const float k = L > 0.f ? 1.f / L : L == 0.f ? 0.f : __int_as_float(0x7fffffff);
            __nv_bfloat162 a = __floats2bfloat162_rn(x.x * k, x.y * k), b = __floats2bfloat162_rn(x.z * k, x.w * k);
            *reinterpret_cast<uint2*>(p.out + ((size_t)(c.q_start + token) * p.Hq + head) * D + col) =
                make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
        };
        for (int idx = tid; idx < rows * (D / 4); idx += THREADS) {
            const int r = idx / (D / 4), col = (idx - r * (D / 4)) * 4;
            float M = NEG_INF, L = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            float2 ml[WARPS];
#pragma unroll
            for (int k = 0; k < WARPS; ++k) {
                ml[k] = *reinterpret_cast<const float2*>(smem + k * WARP_BYTES + (16 * O_STRIDE + 2 * r) * 4);
                M = fmaxf(M, ml[k].x);
            }
            const float base_m = M == NEG_INF ? 0.f : M;
#pragma unroll
            for (int k = 0; k < WARPS; ++k) {
                const float4 y = *reinterpret_cast<const float4*>(smem + k * WARP_BYTES + (r * O_STRIDE + col) * 4);
                const float f = ex2(ml[k].x - base_m);
                L = fmaf(f, ml[k].y, L);
                x.x = fmaf(f, y.x, x.x); x.y = fmaf(f, y.y, x.y); x.z = fmaf(f, y.z, x.z); x.w = fmaf(f, y.w, x.w);
            }
            if (block0 == block1) {
                store_row(r, col, x, M, L);
            } else {
                const size_t place = place_of(blockIdx.x);
                *reinterpret_cast<float4*>(p.part_o + (place * 16 + r) * D + col) = x;
                if (col == 0) *reinterpret_cast<float2*>(p.part_ml + (place * 16 + r) * 2) = make_float2(M, L);
            }
        }
        if (block0 != block1) {
            __threadfence();
            __syncthreads();
            if (tid == 0) ticket_s = atomicAdd(p.tickets + block0, 1);
            __syncthreads();
            if (ticket_s == block1 - block0) {
                // All pieces have left their sums: they are added in order, whichever block came last.
                __threadfence();
                if (tid == 0) p.tickets[block0] = 0;
                for (int idx = tid; idx < rows * (D / 4); idx += THREADS) {
                    const int r = idx / (D / 4), col = (idx - r * (D / 4)) * 4;
                    float M = NEG_INF, L = 0.f;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int b = block0; b <= block1; ++b) M = fmaxf(M, __ldcg(p.part_ml + (place_of(b) * 16 + r) * 2));
                    const float base_m = M == NEG_INF ? 0.f : M;
#pragma unroll 4
                    for (int b = block0; b <= block1; ++b) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + (place_of(b) * 16 + r) * 2));
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(p.part_o + (place_of(b) * 16 + r) * D + col));
                        const float f = ex2(ml.x - base_m);
                        L = fmaf(f, ml.y, L);
                        x.x = fmaf(f, y.x, x.x); x.y = fmaf(f, y.y, x.y); x.z = fmaf(f, y.z, x.z); x.w = fmaf(f, y.w, x.w);
                    }
                    store_row(r, col, x, M, L);
                }
            }
        }
        __syncthreads();                                     // the slots are the next piece's
    }
}

template <int STORE, bool HALF_ROWS>
static int launch(const Params& p, int blocks, cudaStream_t stream) {
    const size_t smem = WARPS * WARP_BYTES + (size_t)(p.segments + 1) * 4;
    static int configured = -1;                              // the device that has been told of the shared memory
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    if (configured != device) {
        e = cudaFuncSetAttribute(attention_quant_kernel<STORE, HALF_ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 WARPS * WARP_BYTES + (MAX_SEGMENTS + 1) * 4);
        if (e != cudaSuccess) return (int)e;
        configured = device;
    }
    kvb_launch(attention_quant_kernel<STORE, HALF_ROWS>, dim3(blocks), dim3(THREADS), smem, stream, p);
    return kvb_launch_status();
}

}  // namespace aq

// How many blocks fill an SM, and segments a launch takes.
KVB_API int kvb_attention_quant_blocks() { return aq::BLOCKS_PER_SM; }
KVB_API int kvb_attention_quant_max_segments() { return aq::MAX_SEGMENTS; }

// Segments of up to `max_q` tokens (the others' rows stay as they are).  page_size: a power of two from 4 on.  scratch:
// 2 * blocks * 16 * (D + 2) floats; tickets: blocks ints, zero before the first launch (the kernel leaves them zero).
KVB_API int kvb_attention_quant(int store, const void* q, void* out, const void* k_codes, const void* v_codes, const void* k_scales, const void* v_scales,
                                int num_pages, const int* block_table, int table_stride, int segments, int T, const int* seg_q_start,
                                const int* seg_q_len, const int* seg_kv_len, int max_q, int Hq, int Hkv, int page_size, int reach, int keep,
                                const float* sink, const float* slopes, float cap, float scale, float* scratch, int* tickets, int blocks, int min_units,
                                int* err, cudaStream_t stream) {
    using namespace aq;
    if (segments <= 0 || T <= 0) return KVB_OK;
    if (store != KVB_E4M3 && store != KVB_INT8) return KVB_ERR_DTYPE;
    if (Hkv < 1 || Hq % Hkv != 0 || page_size < 4 || (page_size & (page_size - 1)) != 0 || num_pages < 1 || max_q < 1 || keep < 0 || cap < 0.f || blocks < 1 ||
        min_units < 1 || table_stride < 1)
        return KVB_ERR_SHAPE;
    if (segments > MAX_SEGMENTS) return KVB_ERR_LIMIT;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)scratch) & 15) return KVB_ERR_ALIGN;
    if (((uintptr_t)k_scales | (uintptr_t)v_scales) & 3) return KVB_ERR_ALIGN;
    const int group = Hq / Hkv;
    // The line of units is counted in 32 bits.
    const long long tiles = ((long long)T * group) / 16 + segments, units = (long long)table_stride * page_size / UNIT + 3 + PIECE_COST;
    if (tiles * Hkv * units > 0x3fffffffll || (long long)table_stride * page_size > 0x3fffffffll) return KVB_ERR_LIMIT;
    Params p = {(const bf16*)q, (bf16*)out, (const uint8_t*)k_codes, (const uint8_t*)v_codes, (const uint8_t*)k_scales, (const uint8_t*)v_scales, num_pages,
                block_table, table_stride, 0, segments, seg_q_start, seg_q_len, seg_kv_len, max_q, Hq, Hkv, group, reach, keep, scale, cap, sink, slopes,
                scratch, scratch + (size_t)2 * blocks * 16 * D, tickets, min_units, err};
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    const bool half_rows = (long long)max_q * group <= 8;
    if (store == KVB_E4M3) return half_rows ? launch<KVB_E4M3, true>(p, blocks, stream) : launch<KVB_E4M3, false>(p, blocks, stream);
    return half_rows ? launch<KVB_INT8, true>(p, blocks, stream) : launch<KVB_INT8, false>(p, blocks, stream);
}
