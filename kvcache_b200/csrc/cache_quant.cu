// Keys and values of a cache entry in eight bits (csrc/cache_quant.cuh): append, read-back, and attention for the sizes and types
// that csrc/attention_quant.cu does not take.
//
// The reference's cache holds half precision only (src/qwen_kernels.cu:111-126 writes it).
#include "cache_quant.cuh"
#include <type_traits>

using namespace cq;

// ---- append ------------------------------------------------------------------------------------------------------------------
// Rows of `qkv` are [Hq heads | Hkv key heads | Hkv value heads | ...] of D numbers, `row_stride` apart.  A query or key head x
// becomes x / sqrt(mean(x^2) + eps) * w (eps > 0; w: D numbers or null), then its first 2 rot_half numbers are turned by the
// row's angles as pairs (t, t + rot_half); queries are rounded to q_out, keys and values quantised into the page of the row's position.
// Keys and values are made in float64 from the inputs (a few operations a number, of rows that are few beside the queries): a code
// is the rounding of the definition's number, whichever kernel writes it, and not of a float32 that lies beside a border.  The scale
// needs the whole row's largest magnitude before the first code is written.
constexpr int APPEND_ROWS = 16;        // rows a block takes at most
struct AppendParams {
    const void* qkv;
    int row_stride;
    const float* bias;         // per column of [q | k | v], or null
    const float* q_norm;
    const float* k_norm;
    float eps;                 // 0: no norm
    const float* cos_t;        // [table_len, rot_half]
    const float* sin_t;
    int rot_half, table_len;
    const int* positions;
    const int* row_segment;
    const int* block_table;
    int table_stride;
    uint8_t* k_codes;          // [num_pages, Hkv, page_size, D]
    uint8_t* v_codes;
    uint8_t* k_scales;         // [num_pages, Hkv, page_size]
    uint8_t* v_scales;
    int num_pages;
    void* q_out;               // [T, Hq * D]
    int T, Hq, Hkv, D, page_size, write_kv;
    int* err;
};

// Where the row's keys lie: index of its slot of head 0 among the pool's rows; -1: no page.
__device__ __forceinline__ long long slot_of(const AppendParams& p, int row, int pos, bool report) {
    const int place = pos / p.page_size;
    const int page = pos >= 0 && place < p.table_stride ? p.block_table[(size_t)p.row_segment[row] * p.table_stride + place] : -1;
    if (page < 0 || page >= p.num_pages) {
        if (report) atomicOr(p.err, KVB_DEV_BAD_PAGE);
        return -1;
    }
    return (long long)page * p.Hkv * p.page_size + pos % p.page_size;
}

// Whether the row's angles are in the table; they are set to the first row's otherwise.
__device__ __forceinline__ size_t angles_of(const AppendParams& p, int pos, bool report) {
    const bool ok = p.rot_half == 0 || (pos >= 0 && pos < p.table_len);
    if (!ok && report) atomicOr(p.err, KVB_DEV_BAD_POS);
    return (size_t)(ok ? pos : 0) * p.rot_half;
}

// Any head size, float32 or bfloat16: a warp a (row, head).  A number is made twice, for the largest and for its code.  F: what the numbers
// are made in.
template <typename F, typename T>
struct HeadNumbers {
    const T* x;
    const float* bias;
    const float* weight;
    const float* cr;
    const float* sr;
    int rot_half;
    bool normed;
    F inv;
    __device__ __forceinline__ F biased(int d) const { return (F)to_f32<T>(x[d]) + (bias ? (F)bias[d] : (F)0); }
    __device__ __forceinline__ F scaled(int d) const { const F v = biased(d); return normed ? (weight ? v * inv * (F)weight[d] : v * inv) : v; }
    __device__ __forceinline__ F at(int d) const {
        const F v = scaled(d);
        if (d >= 2 * rot_half) return v;
        const bool low = d < rot_half;
        const int t = low ? d : d - rot_half;
        const F partner = scaled(low ? d + rot_half : t);
        return low ? v * (F)cr[t] - partner * (F)sr[t] : v * (F)cr[t] + partner * (F)sr[t];
    }
    __device__ __forceinline__ void norm(int D, float eps, int lane) {
        F sum = 0;
        for (int d = lane; d < D; d += 32) { const F v = biased(d); sum += v * v; }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        inv = (F)1 / sqrt(sum / (F)D + (F)eps);
    }
};

template <typename T, int STORE>
__global__ void append_quant_any_kernel(const AppendParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int heads = p.Hq + (p.write_kv ? 2 * p.Hkv : 0), lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (item >= (long long)p.T * heads) return;
    const int row = (int)(item / heads), head = (int)(item - (long long)row * heads), D = p.D;
    const int pos = p.positions[row];
    const bool is_q = head < p.Hq, is_v = head >= p.Hq + p.Hkv;
    const T* x = (const T*)p.qkv + (size_t)row * p.row_stride + (size_t)head * D;
    const float* bias = p.bias ? p.bias + (size_t)head * D : nullptr;
    const size_t angle = angles_of(p, pos, lane == 0);
    const bool normed = !is_v && p.eps > 0.f;
    if (is_q) {
        HeadNumbers<float, T> h = {x, bias, p.q_norm, p.cos_t + angle, p.sin_t + angle, p.rot_half, normed, 1.f};
        if (normed) h.norm(D, p.eps, lane);
        T* out = (T*)p.q_out + ((size_t)row * p.Hq + head) * D;
        for (int d = lane; d < D; d += 32) out[d] = from_f32<T>(h.at(d));
        return;
    }
    HeadNumbers<double, T> h = {x, bias, p.k_norm, p.cos_t + angle, p.sin_t + angle, is_v ? 0 : p.rot_half, normed, 1.0};
    if (normed) h.norm(D, p.eps, lane);
    const long long slot = slot_of(p, row, pos, lane == 0);
    if (slot < 0) return;
    uint32_t top = 0u;
    for (int d = lane; d < D; d += 32) top = max(top, __float_as_uint(__double2float_ru(fabs(h.at(d)))));
    top = __reduce_max_sync(0xffffffffu, top);
    const int byte = scale_byte<STORE>(top);
    const float down = scale_down(byte);
    const long long at = slot + (long long)(is_v ? head - p.Hq - p.Hkv : head - p.Hq) * p.page_size;
    uint8_t* codes = (is_v ? p.v_codes : p.k_codes) + at * D;
    for (int d = lane; d < D; d += 32) codes[d] = down != 0.f ? (uint8_t)code_of<STORE>(h.at(d), down) : (uint8_t)0;
    if (lane == 0) (is_v ? p.v_scales : p.k_scales)[at] = (uint8_t)byte;
}

// bfloat16, heads of 16 LANES numbers, rotated halves in steps of eight: LANES lanes hold a head, eight neighbouring numbers and their eight
// rotation partners each (of what is not rotated, eight numbers of either half).  A block takes `rows` rows, whose pages and angles it looks up
// once, and its groups of lanes go through their heads, with three in flight.
// Bound by latency at sixteen warps an SM (128 registers a thread, which float64 numbers want): schedulers issue in 44 % of the clocks, no pipe is above 25 %
// (float64 4 %), DRAM 18 %, and what warps wait for most are the rows.  2,048 rows of 36 heads of 128 (38 MB in and out) take 10.3 us; eight numbers a lane,
// partners by shuffles, took 16.3, a warp a head with a number a lane 47.
template <int LANES, int STORE, bool NORM>
__global__ void __launch_bounds__(256, 2) append_quant_vec_kernel(const AppendParams p, int rows) {
    constexpr int D = 16 * LANES;
    // [rows][first four cosines, second four, first four sines, second four][eights of rot_half][4]: lanes read neighbouring 16 bytes.
    extern __shared__ __align__(16) float4 angles[];
    __shared__ long long slots[APPEND_ROWS];
    // The rows' metadata and tables are older than the product before this kernel.
    const int row0 = blockIdx.x * rows, lane = threadIdx.x & 31, li = lane & (LANES - 1), half = p.rot_half, eights = half / 8;
    const uint32_t group_mask = ((1u << LANES) - 1u) << (lane & ~(LANES - 1));
    const int groups = blockDim.x / LANES, heads = p.Hq + (p.write_kv ? 2 * p.Hkv : 0), here = min(rows, p.T - row0);
    if ((int)threadIdx.x < here) {
        const int pos = p.positions[row0 + threadIdx.x];
        slots[threadIdx.x] = p.write_kv ? slot_of(p, row0 + threadIdx.x, pos, true) : -1;
        angles_of(p, pos, true);
    }
    for (int i = threadIdx.x; i < here * 4 * eights; i += blockDim.x) {
        const int r = i / (4 * eights), c = (i - r * 4 * eights) / eights, j = i % eights;
        const size_t angle = angles_of(p, p.positions[row0 + r], false) + 8 * j + 4 * (c & 1);
        angles[i] = *reinterpret_cast<const float4*>((c < 2 ? p.cos_t : p.sin_t) + angle);
    }
    // This lane's first numbers, and how far the others lie behind them.
    const bool rotated = li < eights;
    const int d = rotated ? 8 * li : 2 * half + 8 * (li - eights), apart = rotated ? half : (D - 2 * half) / 2;
    pdl_wait();
    pdl_launch_dependents();
    __syncthreads();
    struct Raw { uint4 x, y; };
    auto load = [&](int row, int head) -> Raw {
        if (row >= here) return {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
        const bf16* const from = (const bf16*)p.qkv + (size_t)(row0 + row) * p.row_stride + head * D + d;
        return {*reinterpret_cast<const uint4*>(from), *reinterpret_cast<const uint4*>(from + apart)};
    };
    auto number = [](const uint4& raw, int k) {
        const uint32_t w = k < 2 ? raw.x : k < 4 ? raw.y : k < 6 ? raw.z : raw.w;
        return __uint_as_float(k & 1 ? w & 0xffff0000u : w << 16);
    };
    auto load8 = [](const float* from, float* to) {
        const float4 x = *reinterpret_cast<const float4*>(from), y = *reinterpret_cast<const float4*>(from + 4);
        to[0] = x.x; to[1] = x.y; to[2] = x.z; to[3] = x.w; to[4] = y.x; to[5] = y.y; to[6] = y.z; to[7] = y.w;
    };
    // (row, head) of this and of the next two turns; `groups` is at most a few rows' heads.
    int row = 0, head = threadIdx.x / LANES;
    auto settle = [&](int& r, int& h) { while (h >= heads) { h -= heads; ++r; } };
    settle(row, head);
    int row1 = row, head1 = head + groups;
    settle(row1, head1);
    int row2 = row1, head2 = head1 + groups;
    settle(row2, head2);
    Raw raw = load(row, head), next = load(row1, head1);
    while (row < here) {
        const Raw after = load(row2, head2);
        const bool is_q = head < p.Hq, is_v = head >= p.Hq + p.Hkv;
        float cs[8], sn[8];
        if (rotated && !is_v) {
            const float4* const at = angles + row * 4 * eights + li;
            const float4 c0 = at[0], c1 = at[eights], s0 = at[2 * eights], s1 = at[3 * eights];
            cs[0] = c0.x; cs[1] = c0.y; cs[2] = c0.z; cs[3] = c0.w; cs[4] = c1.x; cs[5] = c1.y; cs[6] = c1.z; cs[7] = c1.w;
            sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w; sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
        }
        const float* const weight = is_q ? p.q_norm : p.k_norm;
        // The numbers as F, biased, normalised and turned.
        auto make = [&](auto* x, auto* y) {
            using F = std::remove_reference_t<decltype(*x)>;
#pragma unroll
            for (int k = 0; k < 8; ++k) { x[k] = (F)number(raw.x, k); y[k] = (F)number(raw.y, k); }
            if (p.bias) {
                float b[8];
                load8(p.bias + (size_t)head * D + d, b);
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] += (F)b[k];
                load8(p.bias + (size_t)head * D + d + apart, b);
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] += (F)b[k];
            }
            if (is_v) return;
            if (NORM) {
                F sum = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) { sum += x[k] * x[k]; sum += y[k] * y[k]; }
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(group_mask, sum, o);
                const F inv = (F)1 / sqrt(sum / D + (F)p.eps);
#pragma unroll
                for (int k = 0; k < 8; ++k) { x[k] *= inv; y[k] *= inv; }
                if (weight) {
                    float w[8];
                    load8(weight + d, w);
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] *= (F)w[k];
                    load8(weight + d + apart, w);
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k] *= (F)w[k];
                }
            }
            if (rotated)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const F c = (F)cs[k], s = (F)sn[k], old = x[k];
                    x[k] = old * c - y[k] * s;
                    y[k] = y[k] * c + old * s;
                }
        };
        if (is_q) {
            float x[8], y[8];
            make(x, y);
            uint32_t out[2][4];
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                __nv_bfloat162 u = __floats2bfloat162_rn(x[k], x[k + 1]), v = __floats2bfloat162_rn(y[k], y[k + 1]);
                out[0][k >> 1] = *reinterpret_cast<uint32_t*>(&u);
                out[1][k >> 1] = *reinterpret_cast<uint32_t*>(&v);
            }
            bf16* const to = (bf16*)p.q_out + ((size_t)(row0 + row) * p.Hq + head) * D + d;
            *reinterpret_cast<uint4*>(to) = make_uint4(out[0][0], out[0][1], out[0][2], out[0][3]);
            *reinterpret_cast<uint4*>(to + apart) = make_uint4(out[1][0], out[1][1], out[1][2], out[1][3]);
        } else {
            double x[8], y[8];
            make(x, y);
            uint32_t top = 0u;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                top = max(top, max(__float_as_uint(__double2float_ru(fabs(x[k]))), __float_as_uint(__double2float_ru(fabs(y[k])))));
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(group_mask, top, o));
            const long long slot = slots[row];
            if (slot >= 0) {
                const int byte = scale_byte<STORE>(top);
                const float down = scale_down(byte);
                uint32_t codes[4] = {0u, 0u, 0u, 0u};
                if (down != 0.f)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        codes[k >> 2] |= code_of<STORE>(x[k], down) << (8 * (k & 3));
                        codes[2 + (k >> 2)] |= code_of<STORE>(y[k], down) << (8 * (k & 3));
                    }
                const long long at = slot + (long long)(is_v ? head - p.Hq - p.Hkv : head - p.Hq) * p.page_size;
                uint8_t* const to = (is_v ? p.v_codes : p.k_codes) + at * D + d;
                *reinterpret_cast<uint2*>(to) = make_uint2(codes[0], codes[1]);
                *reinterpret_cast<uint2*>(to + apart) = make_uint2(codes[2], codes[3]);
                if (li == 0) (is_v ? p.v_scales : p.k_scales)[at] = (uint8_t)byte;
            }
        }
        row = row1; head = head1; raw = next;
        row1 = row2; head1 = head2; next = after;
        head2 += groups;
        settle(row2, head2);
    }
}

template <int LANES>
static int append_vec(const AppendParams& p, int store, cudaStream_t stream) {
    // A group of lanes a head; a block a row, or as many rows as leave no more blocks than the SMs hold at once (with four rows a
    // block 2,048 rows were 512 blocks and took 24 us).
    const int heads = p.Hq + (p.write_kv ? 2 * p.Hkv : 0), wanted = (heads * LANES + 31) / 32 * 32, at_once = 2 * kvb_sm_count();
    const int rows = (p.T + at_once - 1) / at_once < APPEND_ROWS ? (p.T + at_once - 1) / at_once : APPEND_ROWS;
    const dim3 grid((p.T + rows - 1) / rows), block(wanted < 256 ? wanted : 256);
    const size_t smem = (size_t)rows * 2 * p.rot_half * sizeof(float);
    if (store == KVB_E4M3) {
        if (p.eps > 0.f) kvb_launch(append_quant_vec_kernel<LANES, KVB_E4M3, true>, grid, block, smem, stream, p, rows);
        else kvb_launch(append_quant_vec_kernel<LANES, KVB_E4M3, false>, grid, block, smem, stream, p, rows);
    } else {
        if (p.eps > 0.f) kvb_launch(append_quant_vec_kernel<LANES, KVB_INT8, true>, grid, block, smem, stream, p, rows);
        else kvb_launch(append_quant_vec_kernel<LANES, KVB_INT8, false>, grid, block, smem, stream, p, rows);
    }
    return kvb_launch_status();
}

template <typename T>
static int append_any(const AppendParams& p, int store, cudaStream_t stream) {
    const long long items = (long long)p.T * (p.Hq + (p.write_kv ? 2 * p.Hkv : 0));
    const dim3 grid((unsigned)((items + 7) / 8));
    if (store == KVB_E4M3) kvb_launch(append_quant_any_kernel<T, KVB_E4M3>, grid, dim3(256), 0, stream, p);
    else kvb_launch(append_quant_any_kernel<T, KVB_INT8>, grid, dim3(256), 0, stream, p);
    return kvb_launch_status();
}

KVB_API int kvb_append_quant(int dtype, int store, const void* qkv, int row_stride, const float* bias, const float* q_norm, const float* k_norm,
                             float eps, const float* cos_t, const float* sin_t, int rot_half, int table_len, const int* positions,
                             const int* row_segment, const int* block_table, int table_stride, void* k_codes, void* v_codes, void* k_scales,
                             void* v_scales, int num_pages, void* q_out, int T, int Hq, int Hkv, int D, int page_size, int write_kv, int* err,
                             cudaStream_t stream) {
    if (T <= 0) return KVB_OK;
    if (store != KVB_E4M3 && store != KVB_INT8) return KVB_ERR_DTYPE;
    if (D < 1 || Hq < 0 || Hkv < 1 || page_size < 1 || rot_half < 0 || 2 * rot_half > D || num_pages < 1) return KVB_ERR_SHAPE;
    if (row_stride < (Hq + (write_kv ? 2 * Hkv : 0)) * D || (rot_half > 0 && (!cos_t || !sin_t))) return KVB_ERR_SHAPE;
    if ((long long)T * (Hq + 2 * Hkv) > 0x7fffffffll) return KVB_ERR_LIMIT;
    if (Hq + (write_kv ? 2 * Hkv : 0) == 0) return KVB_OK;
    const AppendParams p = {qkv, row_stride, bias, q_norm, k_norm, eps, cos_t, sin_t, rot_half, table_len, positions, row_segment, block_table,
                            table_stride, (uint8_t*)k_codes, (uint8_t*)v_codes, (uint8_t*)k_scales, (uint8_t*)v_scales, num_pages, q_out, T, Hq, Hkv, D,
                            page_size, write_kv, err};
    const uintptr_t addresses = (uintptr_t)qkv | (uintptr_t)bias | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)cos_t | (uintptr_t)sin_t |
                                (uintptr_t)q_out | (uintptr_t)k_codes | (uintptr_t)v_codes;
    if (dtype == KVB_BF16 && (addresses & 15) == 0 && row_stride % 8 == 0 && rot_half % 8 == 0) {
        if (D == 64) return append_vec<4>(p, store, stream);
        if (D == 128) return append_vec<8>(p, store, stream);
        if (D == 32) return append_vec<2>(p, store, stream);
        if (D == 256) return append_vec<16>(p, store, stream);
    }
    if (dtype == KVB_BF16) return append_any<bf16>(p, store, stream);
    if (dtype == KVB_F32) return append_any<float>(p, store, stream);
    return KVB_ERR_DTYPE;
}

// ---- read-back ---------------------------------------------------------------------------------------------------------------
// Blocks of 64 keys of every segment, one segment after the other.  ranges: int32 [S + 1, 3] - the blocks before the segment's, and
// its blocks: 0 .. kept - 1, then from `first` on (kernels/cache_plan.py).  Block i becomes page i of k_out / v_out [n, Hkv, 64, D], and
// out_table[segment, block] = i.  Keys that no row of the segment sees (behind its end; before the first row's window, unless among the
// first `keep`) become zeros, whatever their pages hold.
// `for_scores`: for a kernel that multiplies weights of zero, too, by values - a token whose key or value is not finite then gets a key of NaN,
// which no row meets that does not see the token, and a value of zeros.
// Attention looks pages up, and where it can fetches keys of earlier steps, before it waits, since elsewhere no kernel of the step in front of it
// writes them.  Here one does: attention over what is read back is told to wait first (PagedKVView.made), for only a wait makes these writes
// visible, not that every block has ended.  `early`: it may then be placed early, too (509 rows of 28 heads of 128 behind 8,192 keys, with append and
// attention: 87 us, 90 otherwise).
constexpr int READ_BLOCK = 64;
struct ExpandParams {
    const uint8_t* k_codes;
    const uint8_t* v_codes;
    const uint8_t* k_scales;
    const uint8_t* v_scales;
    int num_pages;
    const int* block_table;
    int table_stride, page_size;
    const int* ranges;
    int segments;
    const int* seg_q_len;
    const int* seg_kv_len;
    int reach, keep, early;
    void* k_out;
    void* v_out;
    int* out_table;
    int out_stride, Hkv, D, for_scores;
    int* err;
};
// What multiplies the codes of the pool's row `at`.
__device__ __forceinline__ float read_scale(const ExpandParams& p, bool values, long long at) {
    const int byte = (values ? p.v_scales : p.k_scales)[at];
    if (!p.for_scores) return scale_up(byte);
    const bool broken = byte == NOT_FINITE || (values ? p.k_scales : p.v_scales)[at] == NOT_FINITE;
    return broken ? (values ? 0.f : __int_as_float(0x7fffffff)) : scale_up(byte);
}

// The segment that block i belongs to, and which of its blocks it is.
__device__ __forceinline__ void find_block(const ExpandParams& p, int i, int& seg, int& block) {
    int lo = 0;
    for (int hi = p.segments; hi - lo > 1;) { const int mid = (lo + hi) >> 1; if (p.ranges[3 * mid] <= i) lo = mid; else hi = mid; }
    const int j = i - p.ranges[3 * lo], kept = p.ranges[3 * lo + 1];
    seg = lo;
    block = j < kept ? j : p.ranges[3 * lo + 2] + j - kept;
}

template <typename T, int STORE>
__global__ void expand_any_kernel(const ExpandParams p) {
    pdl_wait();
    if (p.early) pdl_launch_dependents();
    const int i = blockIdx.x, hk = blockIdx.y, D = p.D;
    const bool values = blockIdx.z == 1;
    int seg, block;
    find_block(p, i, seg, block);
    const int kv_len = p.seg_kv_len[seg], lo = first_seen_key(kv_len - p.seg_q_len[seg], p.reach), keep = p.reach > 0 ? p.keep : 0;
    if (hk == 0 && !values && threadIdx.x == 0 && block < p.out_stride) p.out_table[(size_t)seg * p.out_stride + block] = i;
    const uint8_t* codes = values ? p.v_codes : p.k_codes;
    T* out = (T*)(values ? p.v_out : p.k_out) + ((size_t)i * p.Hkv + hk) * READ_BLOCK * D;
    const int lane = threadIdx.x & 31;
    for (int r = threadIdx.x >> 5; r < READ_BLOCK; r += blockDim.x >> 5) {
        const int key = block * READ_BLOCK + r;
        long long at = -1;
        if (key < kv_len && (key >= lo || key < keep)) {
            const int place = key / p.page_size;
            const int page = place < p.table_stride ? p.block_table[(size_t)seg * p.table_stride + place] : -1;
            if (page >= 0 && page < p.num_pages) at = ((long long)page * p.Hkv + hk) * p.page_size + key % p.page_size;
            else if (lane == 0) atomicOr(p.err, KVB_DEV_BAD_PAGE);
        }
        const float up = at >= 0 ? read_scale(p, values, at) : 0.f;
        for (int d = lane; d < D; d += 32)
            out[(size_t)r * D + d] = from_f32<T>(at >= 0 ? code_value<STORE>(codes[at * D + d]) * up : 0.f);
    }
}

// Heads in steps of eight numbers: a thread reads eight codes and writes eight numbers, four at a time in flight.
template <typename T> __device__ __forceinline__ void store8(T* to, const float* x);
template <> __device__ __forceinline__ void store8<float>(float* to, const float* x) {
    *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(to + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <> __device__ __forceinline__ void store8<bf16>(bf16* to, const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        __nv_bfloat162 y = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
        w[k] = *reinterpret_cast<uint32_t*>(&y);
    }
    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int STORE>
__global__ void __launch_bounds__(256) expand_vec_kernel(const ExpandParams p) {
    const int i = blockIdx.x, hk = blockIdx.y, D = p.D, chunks = D >> 3;
    int seg, block;
    find_block(p, i, seg, block);
    const int kv_len = p.seg_kv_len[seg], lo = first_seen_key(kv_len - p.seg_q_len[seg], p.reach), keep = p.reach > 0 ? p.keep : 0;
    const int* const table = p.block_table + (size_t)seg * p.table_stride;
    const size_t out = ((size_t)i * p.Hkv + hk) * READ_BLOCK * D;
    constexpr int FLIGHT = 4;                                // of keys and of values each
    bool waited = false;
    for (int c0 = threadIdx.x; c0 < READ_BLOCK * chunks; c0 += FLIGHT * 256) {
        long long at[FLIGHT];
        uint2 code[2][FLIGHT];
        float up[2][FLIGHT];
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) {
            const int c = c0 + f * 256, r = c / chunks, key = block * READ_BLOCK + r;
            at[f] = -1;
            if (c < READ_BLOCK * chunks && key < kv_len && (key >= lo || key < keep)) {
                const int place = key / p.page_size;
                const int page = place < p.table_stride ? table[place] : -1;
                if (page >= 0 && page < p.num_pages) at[f] = ((long long)page * p.Hkv + hk) * p.page_size + key % p.page_size;
                else atomicOr(p.err, KVB_DEV_BAD_PAGE);
            }
        }
        if (!waited) {                                       // up to here only what the step brought along
            waited = true;
            pdl_wait();
            if (p.early) pdl_launch_dependents();
            if (hk == 0 && threadIdx.x == 0 && block < p.out_stride) p.out_table[(size_t)seg * p.out_stride + block] = i;
        }
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) {
            code[0][f] = code[1][f] = make_uint2(0u, 0u);
            up[0][f] = up[1][f] = 0.f;
            if (at[f] >= 0) {
                const size_t from = at[f] * D + ((c0 + f * 256) % chunks) * 8;
                code[0][f] = *reinterpret_cast<const uint2*>(p.k_codes + from);
                code[1][f] = *reinterpret_cast<const uint2*>(p.v_codes + from);
                up[0][f] = read_scale(p, false, at[f]);
                up[1][f] = read_scale(p, true, at[f]);
            }
        }
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) {
            const int c = c0 + f * 256;
            if (c >= READ_BLOCK * chunks) break;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                float x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = code_value<STORE>(((k < 4 ? code[v][f].x : code[v][f].y) >> (8 * (k & 3))) & 255u) * up[v][f];
                store8<T>((T*)(v ? p.v_out : p.k_out) + out + (size_t)c * 8, x);
            }
        }
    }
}

template <typename T>
static int expand(const ExpandParams& p, int store, int n, cudaStream_t stream) {
    const bool vec = p.D % 8 == 0 && (((uintptr_t)p.k_codes | (uintptr_t)p.v_codes) & 7) == 0 && (((uintptr_t)p.k_out | (uintptr_t)p.v_out) & 15) == 0;
    const dim3 grid(n, p.Hkv, vec ? 1 : 2);
    if (store == KVB_E4M3) kvb_launch(vec ? expand_vec_kernel<T, KVB_E4M3> : expand_any_kernel<T, KVB_E4M3>, grid, dim3(256), 0, stream, p);
    else kvb_launch(vec ? expand_vec_kernel<T, KVB_INT8> : expand_any_kernel<T, KVB_INT8>, grid, dim3(256), 0, stream, p);
    return kvb_launch_status();
}

KVB_API int kvb_cache_expand(int dtype, int store, const void* k_codes, const void* v_codes, const void* k_scales, const void* v_scales, int num_pages,
                             const int* block_table, int table_stride, int page_size, const int* ranges, int segments, int n,
                             const int* seg_q_len, const int* seg_kv_len, int reach, int keep, void* k_out, void* v_out, int* out_table, int out_stride, int Hkv, int D,
                             int for_scores, int early, int* err, cudaStream_t stream) {
    if (n <= 0) return KVB_OK;
    if (store != KVB_E4M3 && store != KVB_INT8) return KVB_ERR_DTYPE;
    if (D < 1 || Hkv < 1 || Hkv > 65535 || page_size < 1 || num_pages < 1 || keep < 0 || segments < 1) return KVB_ERR_SHAPE;
    const ExpandParams p = {(const uint8_t*)k_codes, (const uint8_t*)v_codes, (const uint8_t*)k_scales, (const uint8_t*)v_scales, num_pages, block_table,
                            table_stride, page_size, ranges, segments, seg_q_len, seg_kv_len, reach, keep, early, k_out, v_out, out_table, out_stride, Hkv, D, for_scores, err};
    if (dtype == KVB_BF16) return expand<bf16>(p, store, n, stream);
    if (dtype == KVB_F32) return expand<float>(p, store, n, stream);
    return KVB_ERR_DTYPE;
}

// ---- attention, any size -----------------------------------------------------------------------------------------------------
// One block per (row, query head); the running maximum and sum of csrc/attention_generic.cu over chunks of keys.
#define QUANT_THREADS 128
#define QUANT_MAX_D 1024
struct AttendParams {
    const void* q;
    const uint8_t* k_codes;
    const uint8_t* v_codes;
    const uint8_t* k_scales;
    const uint8_t* v_scales;
    int num_pages;
    const int* block_table;
    int table_stride;
    const int* positions;
    const int* row_segment;
    void* out;
    int Hq, Hkv, D, page_size, reach, keep;
    const float* sink;
    const float* slopes;
    float scale, cap;
    int* err;
};

template <typename T, int STORE>
__global__ void attention_quant_any_kernel(const AttendParams p) {
    pdl_wait();
    pdl_launch_dependents();
    extern __shared__ float smem[];
    const int D = p.D;
    float* q_s = smem;                                      // [D]
    float* p_s = q_s + D;                                   // [QUANT_THREADS]
    long long* at_s = (long long*)(p_s + QUANT_THREADS + (D & 1));   // [QUANT_THREADS] the key's row among the pool's, -1: none
    float* scratch = (float*)(at_s + QUANT_THREADS);        // [33]
    const int r = blockIdx.x, h = blockIdx.y, hk = h / (p.Hq / p.Hkv);
    const int pos = p.positions[r];
    const int* table = p.block_table + (size_t)p.row_segment[r] * p.table_stride;
    const int lo = first_seen_key(pos, p.reach), kept = min(p.reach > 0 ? p.keep : 0, lo), visible = kept + pos - lo + 1;
    const T* qr = (const T*)p.q + ((size_t)r * p.Hq + h) * D;
    for (int d = threadIdx.x; d < D; d += QUANT_THREADS) q_s[d] = to_f32<T>(qr[d]);
    __syncthreads();
    constexpr int DPT = QUANT_MAX_D / QUANT_THREADS;
    float acc[DPT];
#pragma unroll
    for (int i = 0; i < DPT; ++i) acc[i] = 0.f;
    float m = -FLT_MAX, l = 0.f;
    if (p.sink) { m = p.sink[h]; l = 1.f; }
    const float slope = p.slopes ? p.slopes[h] : 0.f;
    for (int base = 0; base < visible; base += QUANT_THREADS) {
        const int i = base + threadIdx.x, j = i < kept ? i : lo + (i - kept);
        float s = -FLT_MAX;
        long long at = -1;
        if (i < visible) {
            const int place = j / p.page_size, page = place < p.table_stride ? table[place] : -1;
            if (page < 0 || page >= p.num_pages) {
                atomicOr(p.err, KVB_DEV_BAD_PAGE);
            } else {
                at = ((long long)page * p.Hkv + hk) * p.page_size + j % p.page_size;
                float dot = 0.f;
                const float up = scale_up(p.k_scales[at]);   // on the codes, exact, not on the sum: that of codes may leave float32 where the key's does not
                for (int d = 0; d < D; ++d) dot = fmaf(q_s[d], code_value<STORE>(p.k_codes[at * D + d]) * up, dot);
                s = dot * p.scale;
                if (p.cap > 0.f) s = p.cap * tanhf(s / p.cap);
                if (p.slopes) s -= slope * (float)(pos - j);
            }
        }
        const float m_new = fmaxf(m, block_max(s, scratch));
        const float corr = expf(m - m_new), weight = at >= 0 ? expf(s - m_new) : 0.f;
        p_s[threadIdx.x] = at >= 0 ? weight * scale_up(p.v_scales[at]) : 0.f;
        at_s[threadIdx.x] = at;
        l = l * corr + block_sum(weight, scratch);          // also orders the writes to p_s and at_s
        m = m_new;
        const int n = min(QUANT_THREADS, visible - base);
#pragma unroll
        for (int i2 = 0; i2 < DPT; ++i2) {
            const int d = threadIdx.x + i2 * QUANT_THREADS;
            if (d < D) {
                float a = acc[i2] * corr;
                for (int t = 0; t < n; ++t)
                    if (at_s[t] >= 0) a = fmaf(p_s[t], code_value<STORE>(p.v_codes[at_s[t] * D + d]), a);
                acc[i2] = a;
            }
        }
        __syncthreads();
    }
    T* out = (T*)p.out + ((size_t)r * p.Hq + h) * D;
#pragma unroll
    for (int i = 0; i < DPT; ++i) {
        const int d = threadIdx.x + i * QUANT_THREADS;
        if (d < D) out[d] = from_f32<T>(l == 0.f ? 0.f : acc[i] / l);
    }
}

KVB_API int kvb_attention_quant_any(int dtype, int store, const void* q, const void* k_codes, const void* v_codes, const void* k_scales,
                                    const void* v_scales, int num_pages, const int* block_table, int table_stride, const int* positions,
                                    const int* row_segment, void* out, int T, int Hq, int Hkv, int D, int page_size, int reach, int keep,
                                    const float* sink, const float* slopes, float cap, float scale, int* err, cudaStream_t stream) {
    if (T <= 0) return KVB_OK;
    if (store != KVB_E4M3 && store != KVB_INT8) return KVB_ERR_DTYPE;
    if (D < 1 || D > QUANT_MAX_D || Hkv < 1 || Hq % Hkv != 0 || Hq > 65535 || page_size < 1 || num_pages < 1 || keep < 0 || cap < 0.f) return KVB_ERR_SHAPE;
    const AttendParams p = {q, (const uint8_t*)k_codes, (const uint8_t*)v_codes, (const uint8_t*)k_scales, (const uint8_t*)v_scales, num_pages, block_table,
                            table_stride, positions, row_segment, out, Hq, Hkv, D, page_size, reach, keep, sink, slopes, scale, cap, err};
    const size_t smem = (size_t)(D + (D & 1) + QUANT_THREADS + 33) * 4 + QUANT_THREADS * 8;
    const dim3 grid(T, Hq);
    if (dtype == KVB_BF16) {
        if (store == KVB_E4M3) kvb_launch(attention_quant_any_kernel<bf16, KVB_E4M3>, grid, dim3(QUANT_THREADS), smem, stream, p);
        else kvb_launch(attention_quant_any_kernel<bf16, KVB_INT8>, grid, dim3(QUANT_THREADS), smem, stream, p);
    } else if (dtype == KVB_F32) {
        if (store == KVB_E4M3) kvb_launch(attention_quant_any_kernel<float, KVB_E4M3>, grid, dim3(QUANT_THREADS), smem, stream, p);
        else kvb_launch(attention_quant_any_kernel<float, KVB_INT8>, grid, dim3(QUANT_THREADS), smem, stream, p);
    } else {
        return KVB_ERR_DTYPE;
    }
    return kvb_launch_status();
}
