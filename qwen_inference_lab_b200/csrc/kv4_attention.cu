// Attention of single tokens over pages of 4 bits (layout: kv4.h) on the CUDA cores, float32 queries and arithmetic.
//
//   out = sum_t p_t (m_t + s_t c_t),  p = softmax over the keys t in (pos - window, pos] of scale q . (m_t + s_t c_t)
//
// One pass with a running maximum and sum.  A block takes one token, one kv head, up to HEADS of the query heads that share it, and a
// span of the context; each of its warps walks every fourth tile of 32 keys.  Scores: a lane owns a key and walks its groups, 16
// bytes of codes at a time (8 keys' bytes are neighbours), q from shared memory, the same word for all lanes.  Values: a lane owns 4
// (or 2 x 4) dimensions and walks the tile's keys; a head of fewer than 128 dimensions has several keys side by side.  Keys that are
// masked or have no page are never read.  Warps merge in shared memory, spans by the last block of a token to arrive, in the
// order of the spans whoever that is.
#include "kv4.h"

static constexpr int WARPS = 4;
static constexpr int TILE = 32;                // keys a warp takes at a time

struct Kv4Singles {
    const float* q;                 // [tokens, q_heads * dim]
    const uint8_t* pages;
    float* out;
    const int* info;                // [n][4]: token, position, table row, longest context of the step
    float* part_o;                  // [n][q_heads][n_spans][dim]
    float* part_ml;                 // [n][q_heads][n_spans][2]
    int* tickets;                   // [n][kv_heads * head chunks], zero between launches
    Kv4Table table;
    int n_spans, q_heads, kv_heads, dim, window;
    float scale_log2;
};

// Quads of 4 dimensions a lane owns: QUADS (2 where dim > 128).
template <int HEADS, int QUADS>
__global__ void __launch_bounds__(32 * WARPS) kv4_singles_kernel(const Kv4Singles a) {
    extern __shared__ float shared[];
    const int dim = a.dim, groups = dim / KV4_GROUP;
    float* qs = shared;                                            // [HEADS][dim]
    float* ps = qs + HEADS * dim;                                  // [WARPS][TILE][HEADS]
    float* merged = ps + WARPS * TILE * HEADS;                     // [WARPS][HEADS][dim]
    float* ml = merged + WARPS * HEADS * dim;                      // [WARPS][HEADS][2]
    __shared__ int last_block;
    qil_wait_for_producer();
    qil_release_consumer();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int share = a.q_heads / a.kv_heads, chunks = (share + HEADS - 1) / HEADS;
    const int kv = blockIdx.y / chunks, chunk = blockIdx.y % chunks, unit = blockIdx.z;
    const int token = a.info[4 * unit], pos = a.info[4 * unit + 1], row = a.info[4 * unit + 2], longest = a.info[4 * unit + 3];
    const int head0 = kv * share + chunk * HEADS, heads = min(HEADS, share - chunk * HEADS);
    const int low = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
    const int reach = a.window > 0 ? min(longest, a.window + TILE - 1) : longest;       // a window begins anywhere in its first tile
    const Kv4Span span = kv4_span(blockIdx.x, a.n_spans, reach, low, pos + 1, TILE);
    if ((int)blockIdx.x >= span.count) return;
    const int page_size = a.table.page_size;
    for (int i = threadIdx.x; i < HEADS * dim; i += 32 * WARPS) {
        const int h = i / dim;
        qs[i] = h < heads ? a.q[((size_t)token * a.q_heads + head0 + h) * dim + i % dim] * a.scale_log2 : 0.f;
    }
    __syncthreads();

    float acc[HEADS][QUADS * 4], most[HEADS], total[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        most[h] = -INFINITY;
        total[h] = 0.f;
#pragma unroll
        for (int i = 0; i < QUADS * 4; ++i) acc[h][i] = 0.f;
    }
    const int lanes_a_key = min(32, dim / 4), side_by_side = dim >= 128 ? 1 : 32 / lanes_a_key;      // 24 lanes of a 96-wide head: one key
    const int my_side = lane / lanes_a_key, my_quad = lane % lanes_a_key;
    const bool owns = my_side < side_by_side;
    float* p = ps + warp * TILE * HEADS;
    for (int k0 = span.first / TILE * TILE + warp * TILE; k0 < span.last; k0 += WARPS * TILE) {
        const int key = k0 + lane;
        const bool seen = key >= span.first && key < span.last;
        const int page = seen ? a.table.page(row, key) : -1;
        float score[HEADS];
#pragma unroll
        for (int h = 0; h < HEADS; ++h) score[h] = page >= 0 ? 0.f : -INFINITY;
        if (page >= 0) {
            const uint8_t* run = a.pages + kv4_run_at(page, 0, kv, key % page_size, a.kv_heads, page_size, groups);
            for (int g = 0; g < groups; ++g) {
                const uint4 codes = *reinterpret_cast<const uint4*>(run + kv4_code_at(g, key));
                const unsigned pair = *reinterpret_cast<const unsigned*>(run + kv4_pair_at(g, key, groups));
                const float s = kv4_step(pair), m = kv4_base(pair);
                const unsigned word[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
                for (int w = 0; w < 4; ++w)
#pragma unroll
                    for (int i = 0; i < 8; i += 4) {
                        float k[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) k[j] = fmaf(s, (float)((word[w] >> (4 * (i + j))) & 15u), m);
#pragma unroll
                        for (int h = 0; h < HEADS; ++h) {
                            const float4 q = *reinterpret_cast<const float4*>(qs + h * dim + g * KV4_GROUP + w * 8 + i);
                            score[h] = fmaf(q.x, k[0], fmaf(q.y, k[1], fmaf(q.z, k[2], fmaf(q.w, k[3], score[h]))));
                        }
                    }
            }
        }
        // a NaN among the scores must reach the sum: fmaxf leaves it out of the maximum, the exponential does not
        __syncwarp();
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            const float peak = fmaxf(most[h], warp_max(score[h]));
            const float against = peak == -INFINITY ? 0.f : peak;
            const float keep = exp2f(most[h] - against);
            most[h] = peak;
            const float e = page >= 0 ? exp2f(score[h] - against) : 0.f;
            total[h] = total[h] * keep + e;
#pragma unroll
            for (int i = 0; i < QUADS * 4; ++i) acc[h][i] *= keep;
            p[lane * HEADS + h] = e;
        }
        __syncwarp();
        for (int j0 = 0; j0 < TILE; j0 += side_by_side) {
            const int j = j0 + my_side;
            const int at = __shfl_sync(0xffffffffu, page, j & 31);
            if (!owns || j >= TILE || at < 0) continue;
            const int slot = (k0 + j) % page_size;
            const uint8_t* run = a.pages + kv4_run_at(at, 1, kv, slot, a.kv_heads, page_size, groups);
#pragma unroll
            for (int n = 0; n < QUADS; ++n) {
                const int quad = my_quad + 32 * n;
                if (4 * quad >= dim) break;
                const int g = quad >> 3;
                const unsigned codes = *reinterpret_cast<const uint16_t*>(run + kv4_code_at(g, slot) + (quad & 7) * 2);
                const unsigned pair = *reinterpret_cast<const unsigned*>(run + kv4_pair_at(g, slot, groups));
                const float s = kv4_step(pair), m = kv4_base(pair);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = fmaf(s, (float)((codes >> (4 * i)) & 15u), m);
#pragma unroll
                    for (int h = 0; h < HEADS; ++h) acc[h][4 * n + i] = fmaf(p[j * HEADS + h], v, acc[h][4 * n + i]);
                }
            }
        }
    }
    // the keys side by side, then the lanes' sums, then the warps
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        total[h] = warp_sum(total[h]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            for (int o = 16; o >= lanes_a_key && side_by_side > 1; o >>= 1) acc[h][i] += __shfl_xor_sync(0xffffffffu, acc[h][i], o);
        if (lane == 0) {
            ml[(warp * HEADS + h) * 2] = most[h];
            ml[(warp * HEADS + h) * 2 + 1] = total[h];
        }
        if (owns && my_side == 0)
#pragma unroll
            for (int n = 0; n < QUADS; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * (my_quad + 32 * n) < dim) merged[(warp * HEADS + h) * dim + 4 * (my_quad + 32 * n) + i] = acc[h][4 * n + i];
    }
    __syncthreads();
    const bool alone = span.count == 1;
    for (int i = threadIdx.x; i < heads * dim; i += 32 * WARPS) {
        const int h = i / dim, d = i % dim;
        float peak = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) peak = fmaxf(peak, ml[(w * HEADS + h) * 2]);
        const float against = peak == -INFINITY ? 0.f : peak;
        float sum = 0.f, l = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float keep = exp2f(ml[(w * HEADS + h) * 2] - against);
            sum += merged[(w * HEADS + h) * dim + d] * keep;
            l += ml[(w * HEADS + h) * 2 + 1] * keep;
        }
        if (alone) {
            a.out[((size_t)token * a.q_heads + head0 + h) * dim + d] = l == 0.f ? 0.f : sum / l;
        } else {
            const size_t slot = ((size_t)unit * a.q_heads + head0 + h) * a.n_spans + blockIdx.x;
            a.part_o[slot * dim + d] = sum;
            if (d == 0) {
                a.part_ml[slot * 2] = peak;
                a.part_ml[slot * 2 + 1] = l;
            }
        }
    }
    if (alone) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        int* ticket = a.tickets + (size_t)unit * gridDim.y + blockIdx.y;
        last_block = atomicAdd(ticket, 1) == span.count - 1;
        if (last_block) *ticket = 0;
    }
    __syncthreads();
    if (!last_block) return;
    __threadfence();
    for (int i = threadIdx.x; i < heads * dim; i += 32 * WARPS) {
        const int h = i / dim, d = i % dim;
        const size_t slot = ((size_t)unit * a.q_heads + head0 + h) * a.n_spans;
        float peak = -INFINITY;
        for (int s = 0; s < span.count; ++s) peak = fmaxf(peak, __ldcg(a.part_ml + (slot + s) * 2));
        const float against = peak == -INFINITY ? 0.f : peak;
        float sum = 0.f, l = 0.f;
        for (int s = 0; s < span.count; ++s) {
            const float keep = exp2f(__ldcg(a.part_ml + (slot + s) * 2) - against);
            sum += __ldcg(a.part_o + (slot + s) * dim + d) * keep;
            l += __ldcg(a.part_ml + (slot + s) * 2 + 1) * keep;
        }
        a.out[((size_t)token * a.q_heads + head0 + h) * dim + d] = l == 0.f ? 0.f : sum / l;
    }
}

template <int HEADS, int QUADS>
static cudaError_t launch_singles(const Kv4Singles& a, int n, cudaStream_t stream) {
    const int share = a.q_heads / a.kv_heads, chunks = (share + HEADS - 1) / HEADS;
    const size_t smem = sizeof(float) * (HEADS * a.dim + WARPS * TILE * HEADS + WARPS * HEADS * a.dim + WARPS * HEADS * 2);
    static QilPerDevice ready;
    const cudaError_t e = ready.once(qil_device(), [] {
        return cudaFuncSetAttribute(kv4_singles_kernel<HEADS, QUADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
    });
    if (e != cudaSuccess) return e;
    return qil_launch_chained(kv4_singles_kernel<HEADS, QUADS>, dim3(a.n_spans, a.kv_heads * chunks, n), dim3(32 * WARPS), smem, stream, a);
}

// Query heads a block takes: the power of two from `share` on, 8 at most (more makes chunks).
static int heads_a_block(int share) { return share >= 5 ? 8 : share >= 3 ? 4 : share; }

extern "C" int qil_kv4_singles_heads(int share) { return heads_a_block(share); }

struct Kv4SinglesCall {
    const void *q, *pages;
    void* out;
    const void* info;
    void *part_o, *part_ml, *tickets;
    const void* block_table;
    cudaStream_t stream;
    float scale;
    int n, n_spans, table_height, table_width, q_heads, kv_heads, dim, page_size, num_pages, window;
};
extern "C" int qil_kv4_singles_call_bytes() { return sizeof(Kv4SinglesCall); }
extern "C" int qil_kv4_singles(const void* packed) {
    const auto [q, pages, out, info, part_o, part_ml, tickets, block_table, stream, scale, n, n_spans, table_height, table_width, q_heads, kv_heads, dim,
                page_size, num_pages, window] = kv4_call<Kv4SinglesCall>(packed);
    if (n <= 0) return 0;
    if (dim <= 0 || dim > KV4_MAX_DIM || dim % KV4_GROUP) QIL_REFUSE("head sizes 32, 64, ..., %d, not %d", KV4_MAX_DIM, dim);
    if (page_size <= 0 || page_size % 8) QIL_REFUSE("pages of a multiple of 8 positions, not %d", page_size);
    if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || n > 65535 || n_spans < 1) QIL_REFUSE("%d query heads, %d kv heads, %d tokens, %d spans", q_heads, kv_heads, n, n_spans);
    const Kv4Singles a = {(const float*)q, (const uint8_t*)pages, (float*)out, (const int*)info, (float*)part_o, (float*)part_ml, (int*)tickets,
                          {(const int*)block_table, table_height, table_width, page_size, num_pages}, n_spans, q_heads, kv_heads, dim, window,
                          scale * 1.4426950408889634f};
    const int heads = heads_a_block(q_heads / kv_heads);
    cudaError_t e = cudaSuccess;
#define KV4_SINGLES(HEADS)                                                                         \
    if (heads == HEADS) e = dim > 128 ? launch_singles<HEADS, 2>(a, n, stream) : launch_singles<HEADS, 1>(a, n, stream)
    KV4_SINGLES(1);
    KV4_SINGLES(2);
    KV4_SINGLES(4);
    KV4_SINGLES(8);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        snprintf(qil_error_text, sizeof(qil_error_text), "%s", cudaGetErrorString(e));
        return (int)e;
    }
    return 0;
}
