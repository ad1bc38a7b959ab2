// Rows into pages of 4 bits and back (layout and rounding: kv4.h).
//
// kv4_store: the tail of a q/k/v projection.  Per head r = 1 / sqrt(mean x^2 + eps), y = x r w (norm), then the first rot_dims
// dimensions turn by the position's angles, (u, v) -> (u c - v s, v c + u s), with u, v half of the rotated dimensions apart or
// neighbours; c, s come from a float32 table or from frequencies (angle = position * frequency in 64 bits: in 32 a position
// beyond 2^17 loses 0.01 rad).  Without weights the norm may come after the turn ("unit heads").  Queries are rounded once to
// their type and written; keys and values are cut into groups and coded.  Keys are computed in 64 bits: which code an element
// gets is a step function of its value, and so is the same here as in any other arithmetic that keeps 64 bits, where in 32 bits one of
// 10^6 elements would land on the other side of a border.  Queries have no borders and stay in 32 bits.
//
// kv4_read: rows of requests as ordinary pages [page][2][kv head][slot][d] of float32 or bfloat16.
#include "kv4.h"

QIL_ERROR_STORAGE

static constexpr int STORE_WARPS = 8;

struct Kv4Store {
    const void* proj;               // T [tokens, ld]; q, k, v from their columns on
    long long ld;
    int q_col, k_col, v_col;
    void* q_out;                    // T [tokens, q_heads * dim]
    uint8_t* pages;
    const void* q_weight;           // W [dim] or null
    const void* k_weight;
    float eps;
    int norm;                       // 0 none, 1 with weights before the turn, 2 without after it
    const float* table;             // [table_rows, rot_dims]: cosines, sines; or null
    int table_rows;
    const float* freq;              // [rot_dims / 2]
    float gain;
    int rot_dims, interleaved;
    const int* positions;
    const int* token_row;
    const int* block_table;
    int table_width, tokens, q_heads, kv_heads, dim, page_size, num_pages;
};

__device__ __forceinline__ double shfl_xor_double(double v, int mask) { return __shfl_xor_sync(0xffffffffu, v, mask); }

// Elements 4 lane .. 4 lane + 3 of a row in every lane; the 8 lanes of a group agree on (s, m).  Returns the codes of the four and
// the pair.
__device__ __forceinline__ void quantise4(const double y[4], unsigned& codes, unsigned& pair) {
    double lo = fmin(fmin(y[0], y[1]), fmin(y[2], y[3])), hi = fmax(fmax(y[0], y[1]), fmax(y[2], y[3]));
    bool good = isfinite(y[0]) && isfinite(y[1]) && isfinite(y[2]) && isfinite(y[3]);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo = fmin(lo, shfl_xor_double(lo, o));
        hi = fmax(hi, shfl_xor_double(hi, o));
    }
    const unsigned votes = __ballot_sync(0xffffffffu, good);
    good = ((votes >> (threadIdx.x & 24)) & 0xffu) == 0xffu;
    const bf16 base = __float2bfloat16_rn(__double2float_rn(lo));
    const bf16 step = __float2bfloat16_rn(__double2float_rn((hi - lo) / 15.0));
    const double m = (double)__bfloat162float(base), s = (double)__bfloat162float(step);
    good = good && isfinite(m) && isfinite(s);
    codes = 0;
    if (good && s > 0.0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) codes |= (unsigned)fmin(fmax(rint((y[i] - m) / s), 0.0), 15.0) << (4 * i);
    }
    pair = good ? ((unsigned)__bfloat16_as_ushort(base) << 16 | __bfloat16_as_ushort(step)) : 0x7fc07fc0u;
}

// Sum over the warp, the same in every lane.
__device__ __forceinline__ double sum_of(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += shfl_xor_double(v, o);
    return v;
}
__device__ __forceinline__ float sum_of(float v) { return warp_sum(v); }

// One head of a token, normed and turned, in arithmetic R; y[q][i] is element 4 (lane + 32 q) + i.
template <typename R, typename T, typename W>
__device__ __forceinline__ void head_row(const Kv4Store& a, const float* __restrict__ x, const R* __restrict__ cs, const W* __restrict__ w,
                                         int lane, R y[2][4]) {
    const int dim = a.dim, half = a.rot_dims >> 1;
    R r = (R)1;
    if (a.norm == 1) {
        R sq = 0;
        for (int j = lane; j < dim; j += 32) sq += (R)x[j] * (R)x[j];
        r = (R)1 / sqrt(sum_of(sq) / (R)dim + (R)a.eps);
    }
    R sq = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 4 * (lane + 32 * q) + i;
            y[q][i] = 0;
            if (d >= dim) continue;
            R own = (R)x[d];
            if (a.norm == 1) own = own * r * (R)to_f32<W>(w[d]);
            if (d < a.rot_dims) {
                const bool second = a.interleaved ? (d & 1) : d >= half;
                const int other = a.interleaved ? (d ^ 1) : (second ? d - half : d + half);
                const int pair = a.interleaved ? d >> 1 : (second ? other : d);
                R partner = (R)x[other];
                if (a.norm == 1) partner = partner * r * (R)to_f32<W>(w[other]);
                const R c = cs[pair], s = cs[half + pair];
                own = second ? own * c + partner * s : own * c - partner * s;
            }
            y[q][i] = own;
            sq += own * own;
        }
    }
    if (a.norm == 2) {
        r = (R)1 / sqrt(sum_of(sq) / (R)dim + (R)a.eps);
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[q][i] *= r;
    }
}

// A block: a token and STORE_WARPS heads, a warp each.
template <typename T, typename W>
__global__ void __launch_bounds__(32 * STORE_WARPS) kv4_store_kernel(const Kv4Store a) {
    __shared__ double angle_d[KV4_MAX_DIM];
    __shared__ float angle_f[KV4_MAX_DIM];
    __shared__ float rows[STORE_WARPS][KV4_MAX_DIM];
    qil_wait_for_producer();
    qil_release_consumer();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, token = blockIdx.x;
    const int pos = a.positions[token], half = a.rot_dims >> 1;
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
        double c, s;
        if (a.table != nullptr) {
            const float* row = a.table + (size_t)min(max(pos, 0), a.table_rows - 1) * a.rot_dims;
            c = row[i];
            s = row[half + i];
        } else {
            sincos((double)pos * (double)a.freq[i], &s, &c);
            c *= (double)a.gain;
            s *= (double)a.gain;
        }
        angle_d[i] = c;
        angle_d[half + i] = s;
        angle_f[i] = (float)c;
        angle_f[half + i] = (float)s;
    }
    __syncthreads();
    const int head = blockIdx.y * STORE_WARPS + warp;
    if (head >= a.q_heads + 2 * a.kv_heads) return;
    const bool is_q = head < a.q_heads, is_k = !is_q && head < a.q_heads + a.kv_heads;
    const int kv = head - a.q_heads - (is_k ? 0 : a.kv_heads);
    const int column = is_q ? a.q_col + head * a.dim : (is_k ? a.k_col : a.v_col) + kv * a.dim;
    const T* src = reinterpret_cast<const T*>(a.proj) + (size_t)token * a.ld + column;
    float* x = rows[warp];
    for (int j = lane; j < a.dim; j += 32) x[j] = to_f32<T>(src[j]);
    __syncwarp();
    if (is_q) {
        float y[2][4];
        head_row<float, T, W>(a, x, angle_f, reinterpret_cast<const W*>(a.q_weight), lane, y);
        T* dst = reinterpret_cast<T*>(a.q_out) + ((size_t)token * a.q_heads + head) * a.dim;
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 4 * (lane + 32 * q) + i;
                if (d < a.dim) dst[d] = from_f32<T>(y[q][i]);
            }
        return;
    }
    double y[2][4];
    if (is_k) {
        head_row<double, T, W>(a, x, angle_d, reinterpret_cast<const W*>(a.k_weight), lane, y);
    } else {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 4 * (lane + 32 * q) + i;
                y[q][i] = d < a.dim ? (double)x[d] : 0.0;
            }
    }
    const int page = kv4_page(a.block_table + (size_t)a.token_row[token] * a.table_width, a.table_width, pos, a.page_size, a.num_pages);
    if (page < 0) return;
    const int slot = pos % a.page_size, groups = a.dim / KV4_GROUP;
    uint8_t* run = a.pages + kv4_run_at(page, is_k ? 0 : 1, kv, slot, a.kv_heads, a.page_size, groups);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        if (128 * q >= a.dim) break;
        unsigned codes, pair;
        quantise4(y[q], codes, pair);
        const int d = 4 * (lane + 32 * q), group = d / KV4_GROUP;
        if (d < a.dim) {
            *reinterpret_cast<uint16_t*>(run + kv4_code_at(group, slot) + (lane & 7) * 2) = (uint16_t)codes;
            if ((lane & 7) == 0) *reinterpret_cast<unsigned*>(run + kv4_pair_at(group, slot, groups)) = pair;
        }
    }
}

extern "C" int qil_kv4_store(const void* proj, long long ld, int q_col, int k_col, int v_col, void* q_out, void* pages,
                             const void* q_weight, const void* k_weight, float eps, int norm, const void* table, int table_rows,
                             const void* freq, float gain, int rot_dims, int interleaved, const void* positions, const void* token_row,
                             const void* block_table, int table_width, int tokens, int q_heads, int kv_heads, int dim, int page_size,
                             int num_pages, int act, int weight, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if (dim <= 0 || dim > KV4_MAX_DIM || dim % KV4_GROUP) QIL_REFUSE("head sizes 32, 64, ..., %d, not %d", KV4_MAX_DIM, dim);
    if (page_size <= 0 || page_size % 8) QIL_REFUSE("pages of a multiple of 8 positions, not %d", page_size);
    if (rot_dims < 0 || rot_dims > dim || rot_dims % 2 || (rot_dims && table == nullptr && freq == nullptr)
        || (table != nullptr && table_rows <= 0))
        QIL_REFUSE("%d rotated dimensions of %d", rot_dims, dim);
    if (q_heads < 0 || kv_heads < 0 || q_heads + kv_heads == 0) QIL_REFUSE("no heads");
    Kv4Store a = {proj, ld, q_col, k_col, v_col, q_out, (uint8_t*)pages, q_weight, k_weight, eps, norm, (const float*)table, table_rows,
                  (const float*)freq, gain, rot_dims, interleaved, (const int*)positions, (const int*)token_row, (const int*)block_table,
                  table_width, tokens, q_heads, kv_heads, dim, page_size, num_pages};
    const dim3 grid(tokens, (q_heads + 2 * kv_heads + STORE_WARPS - 1) / STORE_WARPS);
    QIL_DISPATCH_2(act, weight, qil_launch_chained(kv4_store_kernel<T, W>, grid, dim3(32 * STORE_WARPS), 0, stream, a));
    QIL_CHECK_LAUNCH();
}

// ------------------------------------------------------------------ rows back
__device__ __forceinline__ unsigned two_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
}

// A thread: 8 neighbouring elements (one word of codes) of a position's key or value row.  info: (table row, first position,
// positions, first page of out) a segment; rows of positions without a page are zeros.
static constexpr int READ_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(READ_THREADS)
kv4_read_kernel(const uint8_t* __restrict__ pages, const int* __restrict__ block_table, int table_width, const int* __restrict__ info,
                T* __restrict__ out, int out_pages, int out_page_size, int kv_heads, int dim, int page_size, int num_pages) {
    qil_wait_for_producer();
    qil_release_consumer();
    const int* mine = info + 4 * blockIdx.z;
    const int row = mine[0], first = mine[1], count = mine[2], out_first = mine[3];
    const int words = dim >> 3, groups = dim / KV4_GROUP;
    const int plane = blockIdx.y / kv_heads, head = blockIdx.y % kv_heads;
    const long long at = (long long)blockIdx.x * READ_THREADS + threadIdx.x;
    const int index = (int)(at / words), word = (int)(at % words);
    if (index >= count) return;
    const int out_page = out_first + index / out_page_size;
    if (out_page < 0 || out_page >= out_pages) return;
    const int pos = first + index;
    const int page = kv4_page(block_table + (size_t)row * table_width, table_width, pos, page_size, num_pages);
    float v[8];
    if (page >= 0) {
        const int slot = pos % page_size, group = word >> 2;
        const uint8_t* run = pages + kv4_run_at(page, plane, head, slot, kv_heads, page_size, groups);
        const unsigned codes = *reinterpret_cast<const unsigned*>(run + kv4_code_at(group, slot) + (word & 3) * 4);
        const unsigned pair = *reinterpret_cast<const unsigned*>(run + kv4_pair_at(group, slot, groups));
        const float s = kv4_step(pair), m = kv4_base(pair);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf(s, (float)((codes >> (4 * i)) & 15u), m);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
    T* dst = out + ((((size_t)out_page * 2 + plane) * kv_heads + head) * out_page_size + index % out_page_size) * dim + word * 8;
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(two_bf16(v[0], v[1]), two_bf16(v[2], v[3]), two_bf16(v[4], v[5]), two_bf16(v[6], v[7]));
    } else {
        reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
}

extern "C" int qil_kv4_read(const void* pages, const void* block_table, int table_width, const void* info, int segments, int longest,
                            void* out, int out_pages, int out_page_size, int kv_heads, int dim, int page_size, int num_pages, int act,
                            cudaStream_t stream) {
    if (segments <= 0 || longest <= 0) return 0;
    if (dim <= 0 || dim > KV4_MAX_DIM || dim % KV4_GROUP) QIL_REFUSE("head sizes 32, 64, ..., %d, not %d", KV4_MAX_DIM, dim);
    if (page_size <= 0 || page_size % 8 || out_page_size <= 0) QIL_REFUSE("pages of a multiple of 8 positions, not %d", page_size);
    if (kv_heads <= 0 || 2 * kv_heads > 65535 || segments > 65535) QIL_REFUSE("%d kv heads, %d segments", kv_heads, segments);
    const long long blocks = ((long long)longest * (dim / 8) + READ_THREADS - 1) / READ_THREADS;
    if (blocks > 0x7fffffff) QIL_REFUSE("segments of %d positions", longest);
    const dim3 grid((unsigned)blocks, 2 * kv_heads, segments);
    QIL_DISPATCH_1(act, qil_launch_chained(kv4_read_kernel<T>, grid, dim3(READ_THREADS), 0, stream, (const uint8_t*)pages,
                                           (const int*)block_table, table_width, (const int*)info, (T*)out, out_pages, out_page_size,
                                           kv_heads, dim, page_size, num_pages));
    QIL_CHECK_LAUNCH();
}
