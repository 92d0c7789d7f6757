// Attention of few query rows over cache pages in eight bits (csrc/cache_quant.cuh): single tokens and short portions, bfloat16
// queries and results, compiled per head size with -DKVB_HEAD_DIM=32, 64, 96 or 128.
//
// It computes what the reference's k_batched_paged_decode_attn computes (src/qwen_kernels.cu:293-335), split over keys and merged as
// src/flash_decode.cu:82-101 does, from codes c and exponents e instead of half-precision rows:
//   score_j = scale 2^(e_j) (q . c_j),   out = sum_j w_j 2^(f_j) d_j / sum_j w_j,   w_j = 2^(score_j log2 e)
// with (c, e) a key's and (d, f) a value's row.  The weights that meet the value codes are n_j = 2^(score_j log2 e + f_j - m), m a
// reference that follows the largest of those exponents so far and lags behind it by HEADROOM at most: n_j is at most 2^HEADROOM, and what matters for the sum
// lies near that or 1 whatever the rows' scales are, so that half precision holds it to 2^-11.  The denominator takes n_j 2^(-f_j), in float32.  Scores are products of codes as they are stored
// (mma.sync m16n8k32, a step of which takes half the time of one over half precision) by queries in two parts of eight bits; value codes,
// exact in half precision, meet the weights on mma.sync m16n8k16.
//
// Codes are the operand with 16 rows, S^T = K Q^T and O^T = V^T P^T, so that eight query rows - the heads that share a key head,
// times the tokens of a short portion - fill an MMA, and what a code costs on its way to half precision is paid once for one or two
// eights of rows.  (Queries as the 16 rows: twice the MMAs and sums in registers for seven heads.)
// A warp takes 32 keys at a time - a block's four in turn - and needs nothing from any other until the block's run ends.  The order of an MMA's inner index, and of its
// rows, is free as long as all agree, so a lane's share of a tile is bytes that lie together: for the scores 16 (or 8) of a key's
// numbers, for the sum the same of four neighbouring keys' values.  The warp copies its tiles itself, two ahead (cp.async: 512 bytes
// that lie together with every instruction - with each lane copying what it will read, from 64 bytes a row, the stream alone took 80 us; as
// the kernel is now it takes 63 of 66, the arithmetic alone 47, 64 requests of 28 heads of 128 and 8,192 keys at most), into rows whose 16-byte parts are turned so that neither the
// copies nor the reads meet a bank twice.  No barrier of the block stands in the stream.
//
// Work is shared out by keys: units of 32 keys of every (segment, key head, tile of rows), laid end to end, are cut into equal
// runs, one a block, whatever the lengths.  Where a cut divides a row tile's keys, the pieces' sums meet in scratch, two places a
// block: the last of sixteen neighbours to finish adds them in order, and so on until 32 are left for the last: the same bits whichever is last, and
// none of many pieces waits for one block to read them all (131,072 keys of 4 heads in 103 pieces each: 74 us with one
// block adding all).
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
constexpr int UNIT = 32;                // keys a warp takes at a time
constexpr int KU = D % 64 == 0 ? 16 : 8, KN = D / (4 * KU);                       // bytes a read, reads of a key row by one of the four lanes that share it
constexpr int VU = D % 128 == 0 ? 16 : D % 64 == 0 ? 8 : 4, VN = D / (8 * VU);    // ... of a value row by one of eight
constexpr int K_BYTES = UNIT * D, STAGE_BYTES = 2 * K_BYTES + 64;                 // keys, values, and both scale bytes of a tile
constexpr int STAGES = 2;               // tiles on their way to a warp (three, heads of 64: 14 of them, 64 requests of 8,192 keys at most 30.6 us, two 28.1)
constexpr int O_STRIDE = D + 4;
// A warp's shared memory: its tiles, and over them its sums when a piece ends.
template <int ROW_TILES>
constexpr int warp_bytes = STAGES * STAGE_BYTES > 8 * ROW_TILES * (O_STRIDE * 4 + 8) ? STAGES * STAGE_BYTES : 8 * ROW_TILES * (O_STRIDE * 4 + 8);
// Blocks an SM holds of the kernel for ROW_TILES eights of rows: registers allow 3 of 168 a thread, or 4 of 128, or 2 of 255
// (five of 96, heads of 64, spill: 28.1 to 32.7 us in the case above).  Under these bounds the e4m3 instances spill 28 and 80 bytes (heads of 64, eight and sixteen
// rows), 20 and 64 (128), 0 and 4 (96), the others none.
template <int ROW_TILES> constexpr int blocks_per_sm() { return ROW_TILES == 1 ? (D <= 64 ? 4 : 3) : D <= 64 ? 3 : 2; }
constexpr int MAX_SEGMENTS = 4096;
constexpr int GROUP = 16, MOST = 32;   // pieces whose sums one block adds up: of a group, and of the last ones that are left
constexpr int PIECE_COST = 12;         // what a piece costs beside its keys, in units
constexpr float NEG_INF = -INFINITY;
constexpr float HEADROOM = 8.f;

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
    float* part_o;             // [2 * blocks, rows of a tile, D]
    float* part_ml;            // [2 * blocks, rows of a tile, 2]
    int* tickets;              // [7 * blocks], zero between launches
    int min_units;
    int* err;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool there) {
    const int n = there ? BYTES : 0;                       // the rest is filled with zeros
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(from), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(to), "l"(from), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
template <int BYTES> __device__ __forceinline__ void read_slot(uint32_t from, uint32_t* w) {
    if (BYTES == 16) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(from) : "memory");
    else if (BYTES == 8) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(w[0]), "=r"(w[1]) : "r"(from) : "memory");
    else asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(w[0]) : "r"(from) : "memory");
}
// Where a half tile's numbers lie in shared memory, as a lane sees it.  A row is D bytes in 16-byte parts.  Heads of 128: the eight parts of row
// `key` are turned, part c lies at c ^ 2 ((key / 4) % 4) ^ 4 (key % 2).  Heads of 64: the four parts, c ^ 2 (key / 8), and rows 2 i and 2 i + 1
// change places where key / 4 is odd.  Others: as they come.
struct Lane {
    int copy;        // copy f of 512 bytes: at 512 f + (copy ^ 32 f) with turned parts, else 512 f + copy
    int k;           // key row g, this lane's first part: the next (heads of 128) at k ^ 64, of the others 4 KU further; key row g + 8: 2 D further
    int v[2];        // values of keys 4 t and 4 t + 1; of 4 t + 2 and 4 t + 3: 2 D further
};
__device__ __forceinline__ Lane lane_places(int lane) {
    const int g = lane >> 2, t = lane & 3, key = 4 * (g >> 1) + (g & 1);
    Lane x;
    if (D == 128) {
        x.copy = (lane >> 3) * 128 + (((lane & 7) ^ (4 * ((lane >> 3) & 1))) << 4);
        x.k = key * 128 + ((t ^ (2 * ((g >> 1) & 3)) ^ (4 * (g & 1))) << 4);
        x.v[0] = t * 512 + ((g ^ (2 * t)) << 4);
        x.v[1] = (x.v[0] ^ 64) + 128;
    } else if (D == 64) {
        x.copy = ((lane >> 2) ^ ((lane >> 4) & 1)) * 64 + ((lane & 3) << 4);
        x.k = (key ^ ((g >> 1) & 1)) * 64 + ((t ^ (2 * (g >> 2))) << 4);
        const int at = t * 256 + (((g >> 1) ^ (t & 2)) << 4) + (g & 1) * 8;
        x.v[0] = at + 64 * (t & 1);
        x.v[1] = at + 64 * (1 - (t & 1));
    } else {
        x.copy = lane * 16;
        x.k = key * D + t * KU;
        x.v[0] = t * 4 * D + g * VU;
        x.v[1] = x.v[0] + D;
    }
    return x;
}
__device__ __forceinline__ int copy_place(const Lane& x, int f) { return 512 * f + (D % 64 == 0 && D != 96 ? x.copy ^ (32 * f) : x.copy); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}
// The same for 32 numbers a row in eight bits: codes as they are stored, by queries split in two parts of eight bits.
template <int STORE>
__device__ __forceinline__ void mma8(uint32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2]) {
    if (STORE == KVB_E4M3)
        asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
    else
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}
// Two query numbers (their row's largest lies in 1 .. 2) as two codes of the cache's type each, in the lower two bytes; `joined` is the
// score from their sums.  e4m3: 128 x = high + low / 32, each with four significant bits - all eight of a bfloat16, and what lies 2^-20
// below the row's largest vanishes.  int8: 16320 x = 256 high + low, off by 2^-15 of the row's largest at most.  Either is far below what
// rounds the weights (2^-11).
template <int STORE>
__device__ __forceinline__ void split_queries(float x0, float x1, uint32_t& high, uint32_t& low) {
    if (STORE == KVB_E4M3) {
        const float2 y = make_float2(128.f * x0, 128.f * x1);
        const __nv_fp8x2_storage_t h = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
        const float2 z = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3)));
        high = h;
        low = __nv_cvt_float2_to_fp8x2(make_float2(32.f * (y.x - z.x), 32.f * (y.y - z.y)), __NV_SATFINITE, __NV_E4M3);
    } else {
        const int y0 = __float2int_rn(16320.f * x0), y1 = __float2int_rn(16320.f * x1);      // |y| < 127.5 * 256
        const int h0 = (y0 + 128) >> 8, h1 = (y1 + 128) >> 8;
        high = __byte_perm((uint32_t)h0, (uint32_t)h1, 0x0040) & 0xffffu;
        low = __byte_perm((uint32_t)(y0 - 256 * h0), (uint32_t)(y1 - 256 * h1), 0x0040) & 0xffffu;
    }
}
template <int STORE>
__device__ __forceinline__ float joined(uint32_t high, uint32_t low) {
    if (STORE == KVB_E4M3) return fmaf(__uint_as_float(low), 1.f / 32.f, __uint_as_float(high));
    return (float)(256 * (int)high + (int)low);
}
template <int STORE> constexpr float QUERY_SCALE = STORE == KVB_E4M3 ? 1.f / 128.f : 1.f / 16320.f;
// The 8 x 8 matrix of 16-bit numbers that a warp holds, a row a group of four lanes, turned.
__device__ __forceinline__ uint32_t turned(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
// Two neighbouring codes, the lower or the upper two bytes of a word, as half precision.  An int8 code with its sign bit flipped becomes the
// low bits of 1024 + c + 128.  (e4m3: two conversions take 6 clocks a word and scheduler, putting exponent and mantissa where half
// precision has them by shifts and masks 10.)
template <int STORE>
__device__ __forceinline__ void halves(uint32_t w, uint32_t& lower, uint32_t& upper) {
    if (STORE == KVB_INT8) {
        const uint32_t f = w ^ 0x80808080u, a = __byte_perm(f, 0x64646464u, 0x4140), b = __byte_perm(f, 0x64646464u, 0x4342);
        const __half2 off = __half2half2(__ushort_as_half(0x6480));          // 1152
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off), y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
        lower = *reinterpret_cast<const uint32_t*>(&x);
        upper = *reinterpret_cast<const uint32_t*>(&y);
    } else {
        asm("{.reg .b16 x, y; mov.b32 {x, y}, %2; cvt.rn.f16x2.e4m3x2 %0, x; cvt.rn.f16x2.e4m3x2 %1, y;}" : "=r"(lower), "=r"(upper) : "r"(w));
    }
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
template <int ROWS>
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
    c.row_tiles = (c.q_len * p.group + ROWS - 1) / ROWS;
    return c;
}

template <int STORE, int ROW_TILES>
__global__ void __launch_bounds__(THREADS, blocks_per_sm<ROW_TILES>()) attention_quant_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int ROWS = 8 * ROW_TILES;
    constexpr int WARP_BYTES = warp_bytes<ROW_TILES>;
    int* const first = reinterpret_cast<int*>(smem + WARPS * WARP_BYTES);     // [segments + 1] the line before each segment
    __shared__ int ticket_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

    // Each row tile is cut into equal pieces of at most `share` units, a block a piece, so that none waits for a second: `share` is such that the
    // pieces are no more than the blocks.  Where that leaves the longest piece over a quarter longer, the line of all units, with what a piece
    // costs beside them, is cut into equal runs.
    // first[s]: the pieces, or the line, before segment s.  The step's lengths are metadata that no kernel before this one writes.
    const int blocks = (int)gridDim.x;
    int units = 0, items = 0;
    for (int s = lane; s < p.segments; s += 32) {
        const Segment c = make_segment<ROWS>(p, s);
        items += c.row_tiles * p.Hkv;
        units += c.row_tiles * p.Hkv * c.n;
    }
    units = __reduce_add_sync(0xffffffffu, units);
    items = __reduce_add_sync(0xffffffffu, items);
    const int total = units + items * PIECE_COST;
    const int share_line = (total + blocks - 1) / blocks, share_whole = items < blocks ? (units + blocks - items - 1) / (blocks - items) : units;
    const bool whole = items < blocks && 4 * (long long)share_whole <= 5 * (long long)max(2 * p.min_units, share_line);
    const int share = whole ? max(1, share_whole) : max(2 * p.min_units, share_line);
    // No piece is smaller than a meeting of pieces is worth: none up to 2 min_units, a unit a warp (min_units) where that makes a dozen pieces at
    // most, else two.  One token of 14 heads of 64, smallest piece 4 / 8 / 16 units, us: 200 keys 5.6 / 5.1 / 5.1, 500 6.1 / 6.9 / 7.2, 1,000 5.9 / 6.9 / 8.9,
    // 2,000 6.6 / 6.9 / 9.2, 4,000 8.1 / 7.8 / 9.2; of 28 of 128 6.9 / 6.2 / 6.2, 7.1 / 8.4 / 9.1, 7.7 / 8.2 / 11.2, 9.1 / 9.1 / 11.7, 11.8 / 10.2 / 12.0.
    auto pieces_of = [&](int n) -> int {
        const int size = max(share, n <= 2 * p.min_units ? n : n <= 12 * p.min_units ? p.min_units : 2 * p.min_units);
        return (n + size - 1) / size;
    };
    if (warp == 0) {
        int before = 0;
        for (int base = 0; base < p.segments; base += 32) {
            int sum = 0, mine = 0;
            if (base + lane < p.segments) {
                const Segment c = make_segment<ROWS>(p, base + lane);
                mine = sum = c.row_tiles * p.Hkv * (whole ? pieces_of(c.n) : c.n + PIECE_COST);
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += up; }
            if (base + lane < p.segments) first[base + lane] = before + sum - mine;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) first[p.segments] = before;
    }
    __syncthreads();
    const int line = first[p.segments];
    const int w_begin = (int)min((long long)line, whole ? (long long)blockIdx.x : (long long)blockIdx.x * share), w_end = min(line, w_begin + (whole ? 1 : share));
    int seg = 0;
    for (int hi = p.segments; hi - seg > 1;) { const int mid = (seg + hi) >> 1; if (first[mid] <= w_begin) seg = mid; else hi = mid; }
    bool waited = false;                                     // the first piece's pages are looked up before the kernel in front has ended

    unsigned char* const mine = smem + warp * WARP_BYTES;
    const uint32_t slots = smem_addr(mine);
    const int page_mask = (1 << p.page_shift) - 1;
    const Lane at_lane = lane_places(lane);
    // Rows of an MMA are keys 4 (r / 2) + r % 2 for r < 8, and two further for r + 8: this lane's key rows are g and g + 8 of a tile of
    // 16, its values those of keys 4 t .. 4 t + 3.
    const int key_k = 4 * (g >> 1) + (g & 1);
    // Selectors that put the scale byte of key row g, or g + 8, of four neighbours' into a word's highest byte.
    const uint32_t pick_first = g & 1 ? 0x1444u : 0x0444u, pick_second = g & 1 ? 0x3444u : 0x2444u;

    for (int w = w_begin; w < w_end;) {
        while (first[seg + 1] <= w) ++seg;
        const Segment c = make_segment<ROWS>(p, seg);
        const int off = w - first[seg];
        int item, begin, end, block0, block1;                // a row tile, units of its list, and the blocks that have some of them
        if (whole) {
            const int pieces = pieces_of(c.n), size = (c.n + pieces - 1) / pieces;
            item = off / pieces;
            begin = min(c.n, (off - item * pieces) * size);
            end = min(c.n, begin + size);
            block0 = w - (off - item * pieces);
            block1 = block0 + (c.n + size - 1) / size - 1;
            ++w;
        } else {
            const int per = c.n + PIECE_COST;
            item = off / per;
            const int at = off - item * per, to = min(per, at + w_end - w);
            const int item_first = w - at + PIECE_COST;      // where the row tile's first unit lies in the line
            begin = max(0, at - PIECE_COST);
            end = max(begin, to - PIECE_COST);
            block0 = item_first / share;
            block1 = (item_first + c.n - 1) / share;
            w += to - at;
        }
        if (begin == end) continue;
        const int hk = item / c.row_tiles, row0 = (item - hk * c.row_tiles) * ROWS;
        const int rows = min(ROWS, c.q_len * p.group - row0);
        const bool one = c.q_len == 1;                        // (a division less for each of a single token's rows)
        auto token_of = [&](int row) -> int { return one ? 0 : row / p.group; };
        const int pos_first = c.start + token_of(row0), pos_last = c.start + token_of(row0 + rows - 1);
        const int lo_first = first_seen_key(pos_first, p.reach), lo_last = first_seen_key(pos_last, p.reach);
        const int* const table = p.block_table + (size_t)seg * p.table_stride;

        const int c_keep = c.keep;
        auto key_of = [&](int i) -> int { return (i < c.n_keep ? i : c.tile_begin - c.n_keep + i) * UNIT; };
        // Pages of both halves of a tile, asked for one tile before they are looked at; -1: none that any row sees.  (Pages of fewer than 16
        // tokens are looked up when they are wanted.)
        struct Pages { int of[2]; };
        auto page_of = [&](int key, int keys) -> int {       // of `keys` neighbours from `key` on
            const int place = key >> p.page_shift;
            return key > pos_last || (key + keys <= lo_first && key >= c.keep) || place >= p.table_stride ? -1 : __ldg(table + place);
        };
        auto lookup = [&](int i) -> Pages {
            if (i >= end || p.page_shift < 4) return {{-1, -1}};
            const int key0 = key_of(i);
            return {{page_of(key0, 16), page_of(key0 + 16, 16)}};
        };
        // The pool's row of `key`, which lies in `page`; -1 without one, which is reported if some row sees one of the `keys` from it on.
        auto row_of = [&](int page, int key, int keys) -> int {
            if (page >= 0 && page < p.num_pages) return ((page * p.Hkv + hk) << p.page_shift) + (key & page_mask);
            if (key <= pos_last && (key + keys > lo_first || key < c.keep)) atomicOr(p.err, KVB_DEV_BAD_PAGE);
            return -1;
        };
        // Copies of a tile's keys with both scale bytes, and of its values: one group each.  Keys that no row sees become zeros.
        auto fetch = [&](int i, uint32_t to, const uint8_t* codes, const Pages& pages) {
            const int key0 = key_of(i);
            if (key0 + UNIT - 1 <= pos_last && key0 >= lo_first && (unsigned)pages.of[0] < (unsigned)p.num_pages && (unsigned)pages.of[1] < (unsigned)p.num_pages) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint8_t* const from = codes + (size_t)(((pages.of[s] * p.Hkv + hk) << p.page_shift) + ((key0 + 16 * s) & page_mask)) * D + lane * 16;
#pragma unroll
                    for (int f = 0; f < D / 32; ++f) copy_async(to + s * 16 * D + copy_place(at_lane, f), from + f * 512);
                }
            } else if (p.page_shift >= 4) {                  // edges, pages that are not there
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int half0 = key0 + 16 * s, row = row_of(pages.of[s], half0, 16);
                    const uint8_t* const from = codes + (size_t)max(row, 0) * D + lane * 16;
#pragma unroll
                    for (int f = 0; f < D / 32; ++f) {
                        const int key = half0 + (32 * f + lane) / (D / 16);
                        copy_async<16>(to + s * 16 * D + copy_place(at_lane, f), from + f * 512, row >= 0 && key <= pos_last && (key >= lo_first || key < c_keep));
                    }
                }
            } else {                                         // small pages
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    const int s = c / (D / 32), f = c - s * (D / 32), part = 32 * f + lane, in_half = part / (D / 16), key = key0 + 16 * s + in_half;
                    const int row = row_of(page_of(key, 1), key, 1);
                    const bool seen = row >= 0 && key <= pos_last && (key >= lo_first || key < c_keep);
                    copy_async<16>(to + s * 16 * D + copy_place(at_lane, f), codes + (size_t)max(row, 0) * D + (part - in_half * (D / 16)) * 16, seen);
                }
            }
        };
        auto fetch_keys = [&](int i, int stage, const Pages& pages) {
            if (i < end) {
                const uint32_t to = slots + stage * STAGE_BYTES;
                fetch(i, to, p.k_codes, pages);
                if (lane < 16) {                             // four scale bytes a lane: of the first half's keys and values, then of the second's
                    const int key = key_of(i) + 16 * (lane >> 3) + 4 * (lane & 3);
                    const int row = row_of(p.page_shift >= 4 ? (lane & 8 ? pages.of[1] : pages.of[0]) : page_of(key, 4), key, 4);
                    copy_async<4>(to + 2 * K_BYTES + lane * 4, (lane & 4 ? p.v_scales : p.k_scales) + max(row, 0), row >= 0);
                }
            }
            copies_commit();
        };
        auto fetch_values = [&](int i, int stage, const Pages& pages) {
            if (i < end) fetch(i, slots + stage * STAGE_BYTES + K_BYTES, p.v_codes, pages);
            copies_commit();
        };
        const int mine_first = begin + warp;                 // the warps take tiles in turn
        // Pages are looked up a tile before they are wanted.
        Pages ahead[STAGES + 1];
#pragma unroll
        for (int s = 0; s <= STAGES; ++s) ahead[s] = lookup(mine_first + s * WARPS);
        if (!waited) { waited = true; pdl_wait(); pdl_launch_dependents(); }
        // This lane's numbers of query row 8 j + g: D / 4 of them, KU together.
        constexpr int QN = D / 4 / 8;                        // 16 bytes at a time
        uint4 raw[ROW_TILES][QN];
#pragma unroll
        for (int j = 0; j < ROW_TILES; ++j) {
            const int row = row0 + 8 * j + g, token = token_of(row), head = hk * p.group + row - token * p.group;
            const bf16* const from = p.q + ((size_t)(c.q_start + token) * p.Hq + head) * D + t * KU;
#pragma unroll
            for (int k = 0; k < QN; ++k)
                raw[j][k] = 8 * j + g < rows ? *reinterpret_cast<const uint4*>(from + (k / (KU / 8)) * 4 * KU + (k % (KU / 8)) * 8) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll 1
        for (int s = 0; s < STAGES; ++s) {
            fetch_keys(mine_first + s * WARPS, s, ahead[0]);
            fetch_values(mine_first + s * WARPS, s, ahead[0]);
#pragma unroll
            for (int x = 0; x < STAGES; ++x) ahead[x] = ahead[x + 1];
        }
        Pages next = ahead[0];

        // Queries as fragments, brought to about 1 by a power of two that goes into the score's factor: this lane holds numbers of row
        // 8 j + g, and the scores of rows 8 j + 2 t and the next.
        uint32_t qf[ROW_TILES][2][QN][2];                    // [eight of rows][high or low part][32 numbers of a head]
        float factor[ROW_TILES][2], slope[ROW_TILES][2];
        int pos[ROW_TILES][2], lo[ROW_TILES][2];
        const bool biased = p.cap > 0.f || p.slopes;
#pragma unroll
        for (int j = 0; j < ROW_TILES; ++j) {
            uint32_t top = 0u;
#pragma unroll
            for (int k = 0; k < QN; ++k) {
                const uint32_t x[4] = {raw[j][k].x, raw[j][k].y, raw[j][k].z, raw[j][k].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max(top, max(x[i] & 0x7fffu, (x[i] >> 16) & 0x7fffu));
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = top == 0u || top >= 0x7f80u ? 0 : max(-126, (int)(top >> 7) - 127);
            const float down = __int_as_float(e == 127 ? 0x400000 : (127 - e) << 23), up = top >= 0x7f80u ? __int_as_float(0x7fffffff) : __int_as_float((127 + e) << 23);
#pragma unroll
            for (int k = 0; k < QN; ++k) {
                const uint32_t x[4] = {raw[j][k].x, raw[j][k].y, raw[j][k].z, raw[j][k].w};
                uint32_t high[4], low[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    split_queries<STORE>(__uint_as_float(x[i] << 16) * down, __uint_as_float(x[i] & 0xffff0000u) * down, high[i], low[i]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    qf[j][0][k][i] = high[2 * i] | high[2 * i + 1] << 16;
                    qf[j][1][k][i] = low[2 * i] | low[2 * i + 1] << 16;
                }
            }
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2) {
                const int r = 8 * j + 2 * t + e2, token2 = token_of(row0 + r);
                pos[j][e2] = r < rows ? c.start + token2 : 0;
                lo[j][e2] = first_seen_key(pos[j][e2], p.reach);
                slope[j][e2] = r < rows && p.slopes ? p.slopes[hk * p.group + row0 + r - token2 * p.group] : 0.f;
                factor[j][e2] = p.scale * QUERY_SCALE<STORE> * __shfl_sync(0xffffffffu, up, 4 * (2 * t + e2)) * (biased ? 1.f : 1.4426950408889634f);
            }
        }

        float o[ROW_TILES][VN * VU / 2][4];                  // sums of columns (of this lane's) 2 x and 2 x + 1 for its two rows
        float m[ROW_TILES][2], l[ROW_TILES][2];
#pragma unroll
        for (int j = 0; j < ROW_TILES; ++j) {
#pragma unroll
            for (int i = 0; i < VN * VU / 2; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
            m[j][0] = m[j][1] = NEG_INF;
            l[j][0] = l[j][1] = 0.f;
        }

        float s[2][ROW_TILES][4];                            // scores, then weights: [half][eight of rows][key row g or g + 8, query row]
        // Weights of the tile from `key0` on, whose scale bytes are given, from its scores.  MASKED: some row may miss a key of it, or scores are capped or
        // biased.
        auto weigh = [&](int key0, const uint32_t (&kb)[2], const uint32_t (&vb)[2], auto masked_tag) {
            constexpr bool MASKED = decltype(masked_tag)::value;
            // Exponents of the weights that the value codes get: score (base 2) + the value row's exponent.
            float inv[2][2];
            uint32_t hidden = 0u;                            // (MASKED) a bit a score
            bool above = false;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const uint32_t pick = n ? pick_second : pick_first;
                    const float up = __uint_as_float(__byte_perm(kb[h], 0u, pick) >> 1);                             // byte << 23
                    const float shift = __uint_as_float(__byte_perm(vb[h], 0x4b000000u, 0x7550u | (pick >> 12))) - 8388735.f;      // byte - 127
                    inv[h][n] = __uint_as_float(0x7f000000u - (__byte_perm(vb[h], 0u, pick) >> 1));                  // -infinity for a row that is not finite
                    const int key = key0 + 16 * h + key_k + 2 * n;
#pragma unroll
                    for (int j = 0; j < ROW_TILES; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = s[h][j][2 * n + e];
                            if (MASKED && biased) {
                                x = x * up * factor[j][e];
                                if (p.cap > 0.f) x = p.cap * (1.f - __fdividef(2.f, 1.f + ex2(x / p.cap * 2.885390081777927f)));
                                x = fmaf(x - slope[j][e] * (float)(pos[j][e] - key), 1.4426950408889634f, shift);
                            } else {
                                x = fmaf(x, up * factor[j][e], shift);
                            }
                            if (MASKED && !(key <= pos[j][e] && (key >= lo[j][e] || key < c.keep))) {
                                x = NEG_INF;
                                hidden |= 1u << (((2 * h + n) * ROW_TILES + j) * 2 + e);
                            }
                            s[h][j][2 * n + e] = x;
                            above |= x > m[j][e] + HEADROOM;
                        }
                }
            // The reference that weights are taken against follows a row's maximum only when that has moved by 2^HEADROOM, far below half
            // precision's 2^16: then the row's lanes agree on it and what has been added up is rescaled.
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int j = 0; j < ROW_TILES; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(fmaxf(s[0][j][e], s[0][j][2 + e]), fmaxf(s[1][j][e], s[1][j][2 + e]));
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                        const float now = fmaxf(m[j][e], top);
                        const float corr = ex2(m[j][e] - (now == NEG_INF ? 0.f : now));
                        m[j][e] = now;
                        l[j][e] *= corr;
#pragma unroll
                        for (int i = 0; i < VN * VU / 2; ++i) { o[j][i][e] *= corr; o[j][i][2 + e] *= corr; }
                    }
            }
#pragma unroll
            for (int j = 0; j < ROW_TILES; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float base_m = MASKED && m[j][e] == NEG_INF ? 0.f : m[j][e];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            float& x = s[h][j][2 * n + e];
                            x = ex2(x - base_m);
                            l[j][e] = fmaf(x, MASKED && ((hidden >> (((2 * h + n) * ROW_TILES + j) * 2 + e)) & 1u) ? 0.f : inv[h][n], l[j][e]);
                        }
                }
        };

        int stage = 0;
#pragma unroll 1
        for (int i = mine_first; i < end; i += WARPS) {
            const int key0 = key_of(i);
            const Pages after = lookup(i + (STAGES + 1) * WARPS);
            const uint32_t base = slots + stage * STAGE_BYTES;
            const bool any = key0 <= pos_last && (key0 + UNIT > lo_first || key0 < c.keep);       // else other rows of the segment see it
            uint32_t kb[2], vb[2];
            copies_wait<2 * STAGES - 1>();
            __syncwarp();                                    // all lanes' copies
            if (any) {
                uint32_t part[2][2][ROW_TILES][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int j = 0; j < ROW_TILES; ++j) part[h][x][j][0] = part[h][x][j][1] = part[h][x][j][2] = part[h][x][j][3] = 0u;
                    read_slot<4>(base + 2 * K_BYTES + (8 * h + (g >> 1)) * 4, &kb[h]);
                    read_slot<4>(base + 2 * K_BYTES + (8 * h + 4 + (g >> 1)) * 4, &vb[h]);
                }
#pragma unroll
                for (int u = 0; u < KN; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t word[2][KU / 4];
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            read_slot<KU>(base + h * 16 * D + 2 * n * D + (D == 128 ? at_lane.k ^ (64 * u) : at_lane.k + 4 * KU * u), word[n]);
#pragma unroll
                        for (int k = 0; k < KU / 8; ++k)
#pragma unroll
                            for (int j = 0; j < ROW_TILES; ++j)
#pragma unroll
                                for (int x = 0; x < 2; ++x)
                                    mma8<STORE>(part[h][x][j], word[0][2 * k], word[1][2 * k], word[0][2 * k + 1], word[1][2 * k + 1], qf[j][x][u * (KU / 8) + k]);
                    }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < ROW_TILES; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[h][j][e] = joined<STORE>(part[h][0][j][e], part[h][1][j][e]);
            }
            __syncwarp();                                    // all lanes have read the keys: their place is filled anew, STAGES tiles ahead
            fetch_keys(i + STAGES * WARPS, stage, next);
            if (any) {
                if (!biased && key0 + UNIT - 1 <= pos_first && key0 >= lo_last) weigh(key0, kb, vb, std::false_type{});
                else weigh(key0, kb, vb, std::true_type{});
            }
            copies_wait<2 * STAGES - 1>();
            __syncwarp();
            if (any) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t pf[ROW_TILES][2];
#pragma unroll
                    for (int j = 0; j < ROW_TILES; ++j) {
                        pf[j][0] = turned(pack(s[h][j][0], s[h][j][1]));
                        pf[j][1] = turned(pack(s[h][j][2], s[h][j][3]));
                    }
#pragma unroll
                    for (int u = 0; u < VN; ++u) {
                        uint32_t v[4][VU / 4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) read_slot<VU>(base + K_BYTES + h * 16 * D + (i & 2) * D + at_lane.v[i & 1] + u * 8 * VU, v[i]);
#pragma unroll
                        for (int k = 0; k < VU / 4; ++k)
#pragma unroll
                            for (int x = 0; x < 2; ++x) {        // two columns of four keys
                                uint32_t a[4];
                                halves<STORE>(__byte_perm(v[0][k], v[1][k], x ? 0x7362 : 0x5140), a[0], a[1]);
                                halves<STORE>(__byte_perm(v[2][k], v[3][k], x ? 0x7362 : 0x5140), a[2], a[3]);
#pragma unroll
                                for (int j = 0; j < ROW_TILES; ++j) mma(o[j][u * (VU / 2) + 2 * k + x], a[0], a[1], a[2], a[3], pf[j]);
                            }
                    }
                }
            }
            __syncwarp();
            fetch_values(i + STAGES * WARPS, stage, next);
            next = after;
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        copies_wait<0>();

        // The warps' sums meet in shared memory, over the slots.
        __syncwarp();
        float* const o_s = reinterpret_cast<float*>(mine);
        float* const ml_s = o_s + ROWS * O_STRIDE;
#pragma unroll
        for (int j = 0; j < ROW_TILES; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * j + 2 * t + e;
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], x);
#pragma unroll
                for (int u = 0; u < VN; ++u)
#pragma unroll
                    for (int k = 0; k < VU / 4; ++k) {
                        const float(*const x)[4] = &o[j][u * (VU / 2) + 2 * k];
                        *reinterpret_cast<float4*>(o_s + r * O_STRIDE + 8 * VU * u + VU * g + 4 * k) = make_float4(x[0][e], x[0][2 + e], x[1][e], x[1][2 + e]);
                    }
                if (g == 0) { ml_s[2 * r] = m[j][e]; ml_s[2 * r + 1] = l[j][e]; }
            }
        __syncthreads();
        // A block's places: of a row tile that another block has begun, and of one that it leaves to others.
        auto place_of = [&](int b) -> size_t { return (size_t)2 * b + (b > block0 ? 0 : 1); };
        auto store_row = [&](int r, int col, float4 x, float M, float L) {
            const int row = row0 + r, token = token_of(row), head = hk * p.group + row - token * p.group;
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
                ml[k] = *reinterpret_cast<const float2*>(smem + k * WARP_BYTES + (ROWS * O_STRIDE + 2 * r) * 4);
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
                *reinterpret_cast<float4*>(p.part_o + (place * ROWS + r) * D + col) = x;
                if (col == 0) *reinterpret_cast<float2*>(p.part_ml + (place * ROWS + r) * 2) = make_float2(M, L);
            }
        }
        if (block0 != block1) {
            // Adds what n blocks from b0 on (every `step`th) have left, in order: (row, columns, sums, m, l) go to `put`.  A warp takes its rows by
            // itself, with the loads of CHUNK pieces in flight; little code, which only a few blocks meet, and cold.
            auto add_up = [&](int b0, int n, int step, auto put) {
                constexpr int QUADS = D / 4, AT_ONCE = 32 / QUADS, CHUNK = 8;
#pragma unroll 1
                for (int r0 = warp * AT_ONCE; r0 < rows; r0 += WARPS * AT_ONCE) {
                    const int r = r0 + lane / QUADS, col = lane % QUADS * 4;
                    const bool there = lane < AT_ONCE * QUADS && r < rows;
                    float M = NEG_INF, L = 0.f;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                    for (int k0 = 0; k0 < n; k0 += CHUNK) {
                        float2 ml[CHUNK];
                        float4 y[CHUNK];
#pragma unroll
                        for (int k = 0; k < CHUNK; ++k) {
                            ml[k] = make_float2(NEG_INF, 0.f);
                            y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (there && k0 + k < n) {
                                const size_t at = place_of(b0 + (k0 + k) * step) * ROWS + r;
                                ml[k] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + at);
                                y[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D + col));
                            }
                        }
                        float now = M;
#pragma unroll
                        for (int k = 0; k < CHUNK; ++k) now = fmaxf(now, ml[k].x);
                        const float base_m = now == NEG_INF ? 0.f : now, corr = ex2(M - base_m);
                        M = now;
                        L *= corr;
                        x.x *= corr; x.y *= corr; x.z *= corr; x.w *= corr;
#pragma unroll
                        for (int k = 0; k < CHUNK; ++k) {
                            const float f = ex2(ml[k].x - base_m);
                            L = fmaf(f, ml[k].y, L);
                            x.x = fmaf(f, y[k].x, x.x); x.y = fmaf(f, y[k].y, x.y); x.z = fmaf(f, y[k].z, x.z); x.w = fmaf(f, y[k].w, x.w);
                        }
                    }
                    __syncwarp();                            // all of the row has been read
                    if (there) put(r, col, x, M, L);
                }
            };
            // The last of `of` blocks to raise a ticket, which it sets back.
            auto last_of = [&](int* ticket, int of) -> bool {
                __syncthreads();
                if (tid == 0) {
                    // The barrier orders the block's stores before this, and what the others released before the block's reads.
                    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;\n" : "=r"(ticket_s) : "l"(ticket) : "memory");
                    if (ticket_s == of - 1) *ticket = 0;
                }
                __syncthreads();
                return ticket_s == of - 1;
            };
            // More than MOST pieces are added in groups of GROUP neighbours, the groups' sums (which lie where their first pieces' lay) in groups again.
            bool last = true;
            int step = 1;
            for (; last && (block1 - block0) / step >= MOST; step *= GROUP) {
                const int b0 = block0 + ((int)blockIdx.x - block0) / (step * GROUP) * (step * GROUP);
                const int members = min(GROUP, (block1 - b0) / step + 1);
                // A block leads a group of one item that starts in it and of one that goes through it, of each size.
                last = last_of(p.tickets + ((size_t)(step == 1 ? 0 : step == GROUP ? 1 : 2) * gridDim.x + b0) * 2 + (b0 == block0), members);
                if (last) {
                    float* const to_o = p.part_o + place_of(b0) * ROWS * D;
                    float* const to_ml = p.part_ml + place_of(b0) * ROWS * 2;
                    add_up(b0, members, step, [&](int r, int col, float4 x, float M, float L) {
                        *reinterpret_cast<float4*>(to_o + r * D + col) = x;
                        if (col == 0) *reinterpret_cast<float2*>(to_ml + r * 2) = make_float2(M, L);
                    });
                }
            }
            if (last && last_of(p.tickets + (size_t)6 * gridDim.x + block0, (block1 - block0) / step + 1))
                add_up(block0, (block1 - block0) / step + 1, step, store_row);
        }
        __syncthreads();                                     // the slots are the next piece's
    }
    if (!waited) { pdl_wait(); pdl_launch_dependents(); }    // blocks without work as well: what comes next may count on all before it
}

template <int STORE, int ROW_TILES>
static int launch(Params p, int sms, long long pieces, cudaStream_t stream) {
    const size_t smem = WARPS * warp_bytes<ROW_TILES> + (size_t)(p.segments + 1) * 4;
    static int configured = -1;                              // the device that has been told of the shared memory
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    if (configured != device) {
        e = cudaFuncSetAttribute(attention_quant_kernel<STORE, ROW_TILES>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 WARPS * warp_bytes<ROW_TILES> + (MAX_SEGMENTS + 1) * 4);
        if (e != cudaSuccess) return (int)e;
        configured = device;
    }
    const int blocks = (int)min((long long)sms * blocks_per_sm<ROW_TILES>(), pieces);
    p.part_ml = p.part_o + (size_t)2 * blocks * 8 * ROW_TILES * D;
    kvb_launch(attention_quant_kernel<STORE, ROW_TILES>, dim3(blocks), dim3(THREADS), smem, stream, p);
    return kvb_launch_status();
}

constexpr int MOST_BLOCKS = 4;         // of any of the kernels, on an SM

// Sixteen rows at once where a segment has more than eight.  (Four eights, heads of 64: 37 rows of 14 heads behind 5,000 keys 20.7 us, two 17.6.)
template <int STORE>
static int launch_rows(const Params& p, long long rows, int sms, long long pieces, cudaStream_t stream) {
    return rows <= 8 ? launch<STORE, 1>(p, sms, pieces, stream) : launch<STORE, 2>(p, sms, pieces, stream);
}

}  // namespace aq

// What a launch needs for every SM: tickets, and floats of scratch.
KVB_API int kvb_attention_quant_tickets() { return 7 * aq::MOST_BLOCKS; }
KVB_API int kvb_attention_quant_scratch() {
    using namespace aq;
    const int one = blocks_per_sm<1>() * 8, two = blocks_per_sm<2>() * 16;
    return 2 * (one > two ? one : two) * (D + 2);
}

// Segments of up to `max_q` tokens (the others' rows stay as they are).  page_size: a power of two from 4 on.  scratch and tickets:
// as above for each of `sms` SMs; the tickets zero before the first launch (the kernel leaves them zero).
KVB_API int kvb_attention_quant(int store, const void* q, void* out, const void* k_codes, const void* v_codes, const void* k_scales, const void* v_scales,
                                int num_pages, const int* block_table, int table_stride, int segments, int T, const int* seg_q_start,
                                const int* seg_q_len, const int* seg_kv_len, int max_q, int Hq, int Hkv, int page_size, int reach, int keep,
                                const float* sink, const float* slopes, float cap, float scale, float* scratch, int* tickets, int sms, int min_units,
                                int* err, cudaStream_t stream) {
    using namespace aq;
    if (segments <= 0 || T <= 0) return KVB_OK;
    if (store != KVB_E4M3 && store != KVB_INT8) return KVB_ERR_DTYPE;
    if (Hkv < 1 || Hq % Hkv != 0 || page_size < 4 || (page_size & (page_size - 1)) != 0 || num_pages < 1 || max_q < 1 || keep < 0 || cap < 0.f || sms < 1 ||
        min_units < 1 || table_stride < 1)
        return KVB_ERR_SHAPE;
    if (segments > MAX_SEGMENTS) return KVB_ERR_LIMIT;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)scratch) & 15) return KVB_ERR_ALIGN;
    if (((uintptr_t)k_scales | (uintptr_t)v_scales) & 3) return KVB_ERR_ALIGN;
    const int group = Hq / Hkv;
    // The line of units is counted in 32 bits.
    const long long rows = min((long long)T, (long long)segments * max_q) * group, tiles = rows / 8 + segments, units = (long long)table_stride * page_size / UNIT + 3 + PIECE_COST;
    if (tiles * Hkv * units > 0x3fffffffll || (long long)table_stride * page_size > 0x3fffffffll) return KVB_ERR_LIMIT;
    if ((long long)num_pages * Hkv * page_size > 0x7fffffffll) return KVB_ERR_LIMIT;      // rows of a pool, too
    Params p = {(const bf16*)q, (bf16*)out, (const uint8_t*)k_codes, (const uint8_t*)v_codes, (const uint8_t*)k_scales, (const uint8_t*)v_scales, num_pages,
                block_table, table_stride, 0, segments, seg_q_start, seg_q_len, seg_kv_len, max_q, Hq, Hkv, group, reach, keep, scale, cap, sink, slopes,
                scratch, nullptr, tickets, min_units, err};
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    // Eights of rows a block takes at once go by the longest segment.
    const long long most_rows = (long long)max_q * group;
    if (store == KVB_E4M3) return launch_rows<KVB_E4M3>(p, most_rows, sms, tiles * Hkv * units, stream);
    return launch_rows<KVB_INT8>(p, most_rows, sms, tiles * Hkv * units, stream);
}
