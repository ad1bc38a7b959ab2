// Attention of single tokens and of a few tokens at a time over pages of 4 bits (layout: kv4.h) on mma.sync, bfloat16 queries, for one
// head size (-DQIL_HEAD_DIM=32, 64, ..., 256).
//
//   out = sum_t p_t (m_t + s_t c_t),  p = softmax over the keys t in (pos - window, pos] of scale q . (m_t + s_t c_t)
//
// A block takes a segment's tokens x the query heads of one kv head, up to 8 NT of these rows, and a span of the context; each
// of its four warps walks every fourth tile of 32 keys on its own: 16-byte copies into a ring of stages in shared memory, then
//
//   scores   S^T = K q^T, 16 keys x 8 rows x 16 dimensions a bfloat16 MMA.  A code in the lowest bits of a half word is, read as
//            bfloat16, code 2^-133, and four bits higher code 2^-129: numbers below and in the first binade have one spacing, and an
//            MMA takes them exactly.  So an AND makes an operand of two codes, and a shift two more; a query row carries the power of two
//            that keeps the products normal (and 1/16 where the codes lie higher).  S += s (q . c) in float32, and one MMA more adds
//            sum_g m_g sum(q_g), the sums as three bfloat16 parts each.  Nothing is rounded but the float32 sums.
//   softmax  in the accumulators' layout; the maximum moves when it grew by more than 2^8 (p <= 256 until then, exact algebra)
//   output   O^T = V^T p^T, 16 dimensions x 8 rows x 16 keys an MMA.  The codes go in as above and p carries the power of two (`lift`: 2^118,
//            less where a step was 2 or more).  A weight is two bfloat16 parts, p and what its rounding left, transposed (movmatrix) one by one;
//            times a group's steps that is p s rounded, and beside it (rest s + what that rounding left) rounded, which is off by 2^-15 of p s: two
//            MMAs each, or one where a block has 4 rows at most, since the second parts then take the columns that would be empty.  With two (one) more
//            out = sum c (p s) + sum p m,
//            the bases exact; the sum of p comes from the same MMAs as the last sum.  With p and p s rounded once each the result was off by
//            2.5e-3 of 64 bits where rounding it costs 1.65e-3; now by 1.7e-3.  8 requests of one token behind 8191 (4 rows a block) took 28.2 us with
//            one part, 30.6 with MMAs of their own for the second, 29.5 in the empty columns; 8 of 5 tokens behind 4000 34.3 and 36.4.
//
// What bounds it: with few blocks the chain description -> block table -> first tile, with many the chain of a tile (copy, AND and shift, MMA,
// exponential, transposition, MMA), of which an SM has 16 warps with one tile each under way: 44 % of the issue slots
// and 16 % of the tensor pipe are used.  Instructions still count, since each is a link of that chain.  Other operands
// cost more of them: 128 + c or 1 + c / 16 with the offset taken off afterwards, and e4m3 (a code's byte is code 2^-9), whose MMAs are taken apart into two of 16 bits.
//
// The lanes' keys are permuted (row r of a tile of 8: key r / 2 + 4 (r & 1)) so that the two keys that a register of the second product
// pairs are c and c + 4.  Every read of shared memory is free of bank conflicts.
//
// Keys that a row does not see are selected away among the scores.  Their values take part with weight zero, so groups of values that
// are NaN are set to zero, and the rows that do see them are marked: their outputs of that group are NaN.
//
// Warps merge in shared memory.  Spans merge in their order: as a cluster every block joins a part of the rows out of the shared memory of
// all (1.1 us of 8 spans), beyond a cluster's size the last block to arrive joins what the others left in memory (3.4).
#include "kv4.h"

QIL_ERROR_STORAGE

#ifndef QIL_HEAD_DIM
#define QIL_HEAD_DIM 128
#endif
#define D QIL_HEAD_DIM
static_assert(D % KV4_GROUP == 0 && D >= 32 && D <= KV4_MAX_DIM, "head sizes 32, 64, ..., 256");
static constexpr int G = D / KV4_GROUP, RUN = 160 * G;
static constexpr int WARPS = 4, TILE = 32, STAGES = 2;
static constexpr int STAGE_BYTES = 8 * RUN;            // 4 runs of keys, 4 of values
static constexpr int MOST_SPANS = 128, MOST_CLUSTER = 16;
// The power of two that p carries, p being 256 at most: p 2^118 and p s 2^118 are bfloat16 numbers for steps below 2, and the products with codes
// counted by 2^-133 are normal float32 numbers down to p s = 2^-111.  Larger steps, of which p s 2^lift stays below 2^127 too, lower it.
static constexpr int MOST_LIFT = 118;
static constexpr float NOTHING = -3e38f;               // the largest score of none

struct Kv4Few {
    const bf16* q;                  // [tokens, q_heads * D]
    const uint8_t* pages;
    bf16* out;
    const int* info;                // [n][8]: first token, its position, tokens, table row, tokens of the segments before, longest context of the step
    float* part_o;                  // [few tokens][q_heads][n_spans][D]
    float* part_ml;                 // [few tokens][q_heads][n_spans][2]
    int* tickets;                   // [few tokens][q_heads], zero between launches
    Kv4Table table;
    int n_spans, q_heads, kv_heads, window, most_tokens;
    int clustered;                  // the spans of a tile of rows are a cluster
    int settled;                    // info and the table are older than the kernel before this one
    float scale_log2;
};

// Pure functions of their operands: the compiler may move them.
__device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first product of a sum: nothing to add to.
__device__ __forceinline__ void mma_first(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// The larger of two pairs, half by half; NaN if either is.
__device__ __forceinline__ unsigned max_pairs(unsigned a, unsigned b) {
    unsigned r;
    asm("max.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ unsigned transposed(unsigned v) {
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ unsigned pack_bf16(float low, float high) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ unsigned times_bf16(unsigned a, unsigned b) {
    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const unsigned*>(&v);
}
// a b + c of two pairs each, rounded once.
__device__ __forceinline__ unsigned fma_bf16(unsigned a, unsigned b, unsigned c) {
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&c));
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ unsigned minus_bf16(unsigned a) { return a ^ 0x80008000u; }
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// What lies at an address of this block's shared memory in another block's of the cluster.
__device__ __forceinline__ float cluster_load(unsigned shared_addr, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(map_to_rank(shared_addr, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float2 cluster_load2(unsigned shared_addr, int rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(map_to_rank(shared_addr, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 cluster_load4(unsigned shared_addr, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(map_to_rank(shared_addr, rank)) : "memory");
    return v;
}
// The pairs of a row's groups.
__device__ __forceinline__ void load_pairs(const uint8_t* at, unsigned (&w)[G]) {
    if constexpr (G % 4 == 0) {
#pragma unroll
        for (int g = 0; g < G; g += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(at + 4 * g);
            w[g] = v.x; w[g + 1] = v.y; w[g + 2] = v.z; w[g + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int g = 0; g < G; ++g) w[g] = *reinterpret_cast<const unsigned*>(at + 4 * g);
    }
}

// How many blocks of this kernel share an SM: what the launch bounds ask for.  Of heads of 128 and one tile of rows 4 blocks have 128
// registers a thread and next to no spills; 2 with all the registers they want stream 4.2 TB/s where 4 stream 4.6, 5 spill (2.7; with
// weights of one part each).
constexpr int blocks_a_sm(int nt) { return nt == 1 ? (D <= 128 ? 4 : 2) : (D <= 64 ? 4 : D <= 128 ? 3 : 1); }

// TWICE: up to 4 rows, each in two columns of the MMAs, c and c + 4 alike: the second parts of the products with steps go through the
// second columns, which are added at the end, and take no MMAs of their own.
template <int NT, bool TWICE>
__global__ void __launch_bounds__(32 * WARPS, blocks_a_sm(NT)) kv4_few_kernel(const Kv4Few a) {
    constexpr int ROWS = TWICE ? 4 : 8 * NT;               // of a block
    extern __shared__ __align__(16) unsigned char shared[];
    __shared__ uint4 q_frag[G * NT][32];                   // the second operand of the scores' MMAs, as the lanes hold it
    __shared__ unsigned q_sums[8 * NT][2 * G];             // of a row's groups: the sums' first two parts, the third
    __shared__ float q_unit[8 * NT];                       // what a row's scores are counted in
    __shared__ float row_ml[WARPS][8 * NT][2];
    __shared__ int last_block;
    __shared__ float2 joint_ml[8 * NT];                    // of the block's rows
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int share = a.q_heads / a.kv_heads;
    if (!a.settled) qil_wait_for_producer();                 // 0.9 us of a launch's 4.7 when it is chained to the one before
    const int4 info = reinterpret_cast<const int4*>(a.info)[2 * blockIdx.z];
    const int4 more = reinterpret_cast<const int4*>(a.info)[2 * blockIdx.z + 1];
    const int first_token = info.x, pos0 = info.y, all_rows = info.z * share, longest = more.y;
    const int kv = blockIdx.y, my_span = blockIdx.x % a.n_spans, row0 = blockIdx.x / a.n_spans * ROWS;
    if (row0 >= all_rows || info.z > a.most_tokens) return;            // a segment of more tokens is somebody else's
    const int rows = min(ROWS, all_rows - row0);
    const int pos_low = pos0 + row0 / share, pos_high = pos0 + (row0 + rows - 1) / share;        // of the block's rows
    const int low = a.window > 0 ? max(0, pos_low + 1 - a.window) : 0;
    const int reach = a.window > 0 ? min(longest, a.window + info.z + TILE - 1) : longest;
    const Kv4Span span = kv4_span(my_span, a.n_spans, reach, low, pos_high + 1, TILE);
    if (my_span >= span.count) {
        if (a.clustered && span.count > 1) {                 // the others meet twice
            cluster_sync_all();
            cluster_sync_all();
        }
        return;
    }

    // ---- copies: this warp's tiles are first_tile, first_tile + WARPS, ...
    const int first_tile = span.first / TILE + warp, end_tile = (span.last + TILE - 1) / TILE;
    const int tiles = end_tile > first_tile ? (end_tile - first_tile + WARPS - 1) / WARPS : 0;
    const int page_runs = a.table.page_size >> 3;
    // the number of the run of keys of lane's (tile lane / 4 of eight, run lane % 4) among all runs of the layer, or -1
    auto runs_of = [&](int tile0) -> int {
        const int key = (first_tile + WARPS * (tile0 + (lane >> 2))) * TILE + (lane & 3) * 8;
        if (key >= span.last) return -1;
        const int page = a.table.page(info.w, key);
        return page < 0 ? -1 : (page * 2 * a.kv_heads + kv) * page_runs + (key % a.table.page_size >> 3);
    };
    const unsigned char* ring_at = shared + warp * STAGES * STAGE_BYTES;
    const unsigned ring = (unsigned)__cvta_generic_to_shared(ring_at) + (lane >> 3) * RUN + (lane & 7) * 16;
    int runs_now = tiles ? runs_of(0) : -1, runs_next = tiles > 8 ? runs_of(8) : -1, issued = 0;
    const size_t value_plane = (size_t)a.kv_heads * page_runs * RUN;
    const unsigned char* my_pages = a.pages + (lane & 7) * 16;
    qil_wait_for_producer();
    qil_release_consumer();
    auto issue = [&](int stage) {
        if (issued < tiles) {
            const int run = __shfl_sync(0xffffffffu, runs_now, (issued & 7) * 4 + (lane >> 3));
            const unsigned char* from = my_pages + (size_t)max(run, 0) * RUN;
            const unsigned to = ring + stage * STAGE_BYTES;
            const int bytes = run < 0 ? 0 : 16;             // no page: zeros
#pragma unroll
            for (int i = 0; i < (10 * G + 7) / 8; ++i) {
                if ((10 * G) % 8 == 0 || (lane & 7) + 8 * i < 10 * G) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to + i * 128), "l"(from + i * 128), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to + 4 * RUN + i * 128), "l"(from + value_plane + i * 128), "r"(bytes) : "memory");
                }
            }
            ++issued;
            if ((issued & 7) == 0) {
                runs_now = runs_next;
                runs_next = issued + 8 < tiles ? runs_of(issued + 8) : -1;
            }
        }
        copies_commit();
    };
    unsigned absent = __ballot_sync(0xffffffffu, runs_now < 0);           // of the eight tiles with the one at hand: 4 bits a tile
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(s);

    // ---- queries: a warp a row, a lane 4 neighbouring dimensions (twice beyond 128); times 2^up the row's largest lies in [2^115, 2^116).
    // All of a warp's rows are on their way before the first is looked at: a row takes 0.9 us by itself.
    {
        constexpr int QUADS = (D + 127) / 128, MINE = ROWS / WARPS, COPIES = TWICE ? 2 : 1;
        uint2 word[MINE][QUADS];
#pragma unroll
        for (int j = 0; j < MINE; ++j) {
            const int row = row0 + warp + WARPS * j;
            const bf16* src = a.q + ((size_t)(first_token + row / share) * a.q_heads + kv * share + row % share) * D;
#pragma unroll
            for (int n = 0; n < QUADS; ++n) {
                const int d = 4 * (lane + 32 * n);
                word[j][n] = d < D && row < all_rows ? *reinterpret_cast<const uint2*>(src + d) : make_uint2(0u, 0u);        // nobody's: zeros
            }
        }
#pragma unroll
        for (int j = 0; j < MINE; ++j) {
            const int of = warp + WARPS * j;
            if (j > 0 && row0 + WARPS * j >= all_rows) {        // nobody's, all four of them
                for (int i = lane; i < 4 * G; i += 32) q_frag[(i >> 2) * NT + of / 8][(of & 7) * 4 + (i & 3)] = make_uint4(0u, 0u, 0u, 0u);
                for (int i = lane; i < 2 * G; i += 32) q_sums[of][i] = 0u;
                if (lane == 0) q_unit[of] = 1.f;
                continue;
            }
            float q[QUADS][4], most_q = 0.f;
#pragma unroll
            for (int n = 0; n < QUADS; ++n) {
                const uint2 w = word[j][n];
                q[n][0] = kv4_step(w.x); q[n][1] = kv4_base(w.x); q[n][2] = kv4_step(w.y); q[n][3] = kv4_base(w.y);
#pragma unroll
                for (int i = 0; i < 4; ++i) most_q = fmaxf(most_q, fabsf(q[n][i]));
            }
            most_q = warp_max(most_q);
            const int up = most_q > 0.f && most_q < INFINITY ? 115 - ilogbf(most_q) : 100;
            // 2^up in two factors: it may be beyond float32.  The sums are counted like the products of codes, 2^-133.
            const float up1 = __uint_as_float((unsigned)(127 + up / 2) << 23), up2 = __uint_as_float((unsigned)(127 + up - up / 2) << 23);
#pragma unroll
            for (int n = 0; n < QUADS; ++n) {
                const int d = 4 * (lane + 32 * n), g = d / KV4_GROUP;
#pragma unroll
                for (int i = 0; i < 4; ++i) q[n][i] = q[n][i] * up1 * up2;
                float sum = (q[n][0] + q[n][1]) + (q[n][2] + q[n][3]);
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum = sum * 0x1p-100f * 0x1p-33f;
                if (d < D) {
                    // dimension 8 c + i of the group: of register i % 4 of lane (row, c) the lower half, for i >= 4 the upper one; odd ones meet
                    // codes that lie four bits higher
#pragma unroll
                    for (int copy = of; copy < of + 4 * COPIES; copy += 4) {
                        bf16* to = reinterpret_cast<bf16*>(&q_frag[g * NT + copy / 8][(copy & 7) * 4 + (lane >> 1 & 3)]) + (lane & 1);
                        to[0] = __float2bfloat16_rn(q[n][0]);
                        to[2] = __float2bfloat16_rn(q[n][1] * 0.0625f);
                        to[4] = __float2bfloat16_rn(q[n][2]);
                        to[6] = __float2bfloat16_rn(q[n][3] * 0.0625f);
                        if ((lane & 7) == 0) {
                            const float first = __bfloat162float(__float2bfloat16_rn(sum)), second = __bfloat162float(__float2bfloat16_rn(sum - first));
                            q_sums[copy][2 * g] = pack_bf16(first, second);
                            q_sums[copy][2 * g + 1] = pack_bf16(sum - first - second, 0.f);
                        }
                    }
                }
            }
            // of queries beyond 2^108 a score's unit would be infinite, and infinity times a score of zero
            if (lane < COPIES) q_unit[of + 4 * lane] = fminf(scalbnf(a.scale_log2, 133 - up), 3e38f);
        }
    }
    __syncthreads();
    constexpr int SUMS = (G + 3) / 4;               // MMAs for the bases: four groups each, lane c the parts of group 4 i + c
    uint4 q_reg[NT == 1 ? G : 1];
    unsigned sum_reg[NT][SUMS][2];
    float unit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if constexpr (NT == 1) {
#pragma unroll
            for (int g = 0; g < G; ++g) q_reg[g] = q_frag[g][lane];
        }
#pragma unroll
        for (int i = 0; i < SUMS; ++i) {
            const int g = 4 * i + c;
            sum_reg[nt][i][0] = g < G ? q_sums[nt * 8 + r][2 * min(g, G - 1)] : 0u;
            sum_reg[nt][i][1] = g < G ? q_sums[nt * 8 + r][2 * min(g, G - 1) + 1] : 0u;
        }
        unit[nt][0] = q_unit[nt * 8 + 2 * c];
        unit[nt][1] = q_unit[nt * 8 + 2 * c + 1];
    }

    float acc[NT][G][2][4], side[NT][4];
    // acc times 2^(lift - 133), rows 8 .. 15 2^(lift - 129); side: row g sum(p m), row 8 sum(p)
    // largest scores of rows 2 c, 2 c + 1, in their units: what is taken off a score is one of them, and the largest minus itself is zero
    // however large it is
    float most[NT][2];
    float lift = MOST_LIFT;
    unsigned lift_limit = 128 << 7;                 // a step of that many bits or more (NaN too) asks for another lift
    unsigned marked[NT][2];                     // groups whose values are NaN for them
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[nt][g][0][i] = acc[nt][g][1][i] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) side[nt][i] = 0.f;
        most[nt][0] = most[nt][1] = NOTHING;
        marked[nt][0] = marked[nt][1] = 0u;
    }
    const int order = (r >> 1) + (r & 1) * 4;                     // the key of 8 that row r stands for
    const unsigned half = r & 1 ? 0x7632u : 0x5410u;              // my half of a word of values, of two keys
    auto row_pos = [&](int nt, int i) { return pos0 + min(row0 + (nt * 8 + 2 * c + i) % ROWS, all_rows - 1) / share; };
    const unsigned second = r >= 4 ? ~0u : 0u;                   // TWICE: my column is a second one

    unsigned sink = (127 - MOST_LIFT) << 7 | (127 - MOST_LIFT) << 23;         // 2^-lift, twice
    const unsigned one = r == 0 ? 0x3f803f80u : 0u;
    // tiles of keys that every row sees begin in [plain_low, plain_low + plain_more]
    const int plain_low = max(span.first, a.window > 0 ? pos_high - a.window + 1 : 0);
    const int plain_more = min(pos_low - TILE + 1, span.last - TILE) - plain_low;
    bool far = false;                           // some score is beyond 2^20
    int stage = 0;
    for (int n = 0; n < tiles; ++n) {
        if ((n & 7) == 0 && n > 0) absent = __ballot_sync(0xffffffffu, runs_now < 0);
        issue(stage == 0 ? STAGES - 1 : stage - 1);
        copies_wait<STAGES - 1>();
        __syncwarp();
        const int k0 = (first_tile + WARPS * n) * TILE;
        const unsigned char* keys = ring_at + stage * STAGE_BYTES;
        unsigned char* values = const_cast<unsigned char*>(keys) + 4 * RUN;
        const unsigned gone = absent >> 4 * (n & 7) & 15u;
        // ---- scores [32 keys][8 NT rows] in the rows' units: sc[u][nt][i]: key 16 u + 8 (i / 2) + order, row 8 nt + 2 c + (i & 1)
        float sc[2][NT][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned char* run0 = keys + 2 * u * RUN;
            const unsigned char* run1 = run0 + RUN;
            unsigned pair0[G], pair1[G];
            load_pairs(run0 + 128 * G + order * 4 * G, pair0);
            load_pairs(run1 + 128 * G + order * 4 * G, pair1);
#pragma unroll
            for (int i = 0; i < SUMS; ++i) {
                unsigned base0 = 0u, base1 = 0u;
                if (G % 4 == 0 || 4 * i + c < G) {
                    const unsigned own0 = *reinterpret_cast<const unsigned*>(run0 + 128 * G + order * 4 * G + 16 * i + 4 * c);
                    const unsigned own1 = *reinterpret_cast<const unsigned*>(run1 + 128 * G + order * 4 * G + 16 * i + 4 * c);
                    base0 = __byte_perm(own0, own0, 0x3232);
                    base1 = __byte_perm(own1, own1, 0x3232);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (i == 0) mma_first(sc[u][nt], base0, base1, base0, base1, sum_reg[nt][i][0], sum_reg[nt][i][1]);
                    else mma(sc[u][nt], base0, base1, base0, base1, sum_reg[nt][i][0], sum_reg[nt][i][1]);
                }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const unsigned w0 = *reinterpret_cast<const unsigned*>(run0 + g * 128 + order * 16 + c * 4);
                const unsigned w1 = *reinterpret_cast<const unsigned*>(run1 + g * 128 + order * 16 + c * 4);
                const unsigned w2 = w0 >> 8, w3 = w1 >> 8;
                const float s0 = kv4_step(pair0[g]), s1 = kv4_step(pair1[g]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint4 q = NT == 1 ? q_reg[NT == 1 ? g : 0] : q_frag[g * NT + nt][lane];
                    float dot[4];
                    mma_first(dot, w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, q.x, q.y);
                    mma(dot, w2 & 0x000f000fu, w3 & 0x000f000fu, w2 & 0x00f000f0u, w3 & 0x00f000f0u, q.z, q.w);
                    sc[u][nt][0] = fmaf(s0, dot[0], sc[u][nt][0]);
                    sc[u][nt][1] = fmaf(s0, dot[1], sc[u][nt][1]);
                    sc[u][nt][2] = fmaf(s1, dot[2], sc[u][nt][2]);
                    sc[u][nt][3] = fmaf(s1, dot[3], sc[u][nt][3]);
                }
            }
        }
        // ---- values that are NaN, and a tile with keys that not every row sees
        unsigned* my_pairs = reinterpret_cast<unsigned*>(values + (lane >> 3) * RUN + 128 * G + (lane & 7) * 4 * G);      // of key k0 + lane
        unsigned pairs[G];
        load_pairs(reinterpret_cast<const uint8_t*>(my_pairs), pairs);
        unsigned largest = pairs[0];
#pragma unroll
        for (int g = 1; g < G; ++g) largest = max_pairs(largest, pairs[g]);
        const bool partly = (unsigned)(k0 - plain_low) > (unsigned)plain_more || plain_more < 0 || gone;
        if (partly || __any_sync(0xffffffffu, (largest & 0xffffu) >= lift_limit)) {
            const int key = k0 + lane;
            const bool inside = key >= span.first && key < span.last && !(gone >> (lane >> 3) & 1);
            unsigned nan = 0;
            largest = 0u;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const bool is_nan = !__hbeq2(*reinterpret_cast<const __nv_bfloat162*>(&pairs[g]), *reinterpret_cast<const __nv_bfloat162*>(&pairs[g]));
                if (is_nan) nan |= 1u << g;
                if (!inside || is_nan) my_pairs[g] = 0u;
                else largest = max_pairs(largest, pairs[g]);
            }
            for (unsigned left = __ballot_sync(0xffffffffu, inside && nan != 0); left; left &= left - 1) {
                const int j = __ffs(left) - 1;
                const unsigned groups = __shfl_sync(0xffffffffu, nan, j);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int pos = row_pos(nt, i);
                        if (k0 + j <= pos && (a.window == 0 || k0 + j > pos - a.window)) marked[nt][i] |= groups;
                    }
            }
            // the lift: by the exponent of the tile's largest step, with room for 2^8 of it
            const int exponent = (int)(__reduce_max_sync(0xffffffffu, largest & 0xffffu) >> 7) - 127;
            if (exponent + (int)lift > MOST_LIFT) {
                const int lower = MOST_LIFT - 8 - exponent;
                const float by = scalbnf(1.f, lower - (int)lift);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int g = 0; g < G; ++g)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            acc[nt][g][0][i] *= by;
                            acc[nt][g][1][i] *= by;
                        }
                lift = (float)lower;
                lift_limit = (unsigned)min(MOST_LIFT + 128 - lower, 255) << 7;
                sink = (unsigned)(127 - lower) << 7 | (unsigned)(127 - lower) << 23;
            }
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = k0 + 16 * u + 8 * (i >> 1) + order, pos = row_pos(nt, i & 1);
                        const bool seen = key >= span.first && key < span.last && key <= pos && (a.window == 0 || key > pos - a.window)
                            && !(gone >> (2 * u + (i >> 1)) & 1);
                        if (!seen) sc[u][nt][i] = -INFINITY;
                    }
        }
        unsigned p[2][NT][2], rest[2][NT][2];
        // ---- softmax, and p 2^lift as the second product's operand, as two bfloat16 parts: p[u][nt][i]: keys c, c + 4 of run 2 u + i, row 8 nt + r
        float peak[NT][2];
        bool grew = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                peak[nt][i] = fmaxf(fmaxf(sc[0][nt][i], sc[0][nt][2 + i]), fmaxf(sc[1][nt][i], sc[1][nt][2 + i]));
                grew |= (peak[nt][i] - most[nt][i]) * unit[nt][i] > 8.f;          // the first finite one too
            }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float keep[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float high = peak[nt][i];
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 4));
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 8));
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 16));
                    const bool grow = (high - most[nt][i]) * unit[nt][i] > 8.f;
                    keep[i] = grow ? fast_exp2((most[nt][i] - high) * unit[nt][i]) : 1.f;
                    if (grow) {
                        most[nt][i] = high;
                        far = far || fabsf(high * unit[nt][i]) > 0x1p20f;
                    }
                }
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        acc[nt][g][0][i] *= keep[i & 1];
                        acc[nt][g][1][i] *= keep[i & 1];
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i) side[nt][i] *= keep[i & 1];
            }
            far = __any_sync(0xffffffffu, far);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float minus[2] = {fminf(fmaf(-most[nt][0], unit[nt][0], lift), 3e38f), fminf(fmaf(-most[nt][1], unit[nt][1], lift), 3e38f)};      // finite, of NOTHING too
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    e[i] = fast_exp2(far ? fmaf(sc[u][nt][i] - most[nt][i & 1], unit[nt][i & 1], lift) : fmaf(sc[u][nt][i], unit[nt][i & 1], minus[i & 1]));
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const unsigned first = pack_bf16(e[2 * i], e[2 * i + 1]);
                    p[u][nt][i] = transposed(first);
                    rest[u][nt][i] = transposed(pack_bf16(e[2 * i] - kv4_step(first), e[2 * i + 1] - kv4_base(first)));
                }
            }
        }
        // ---- output
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned char* run0 = values + 2 * u * RUN;
            const unsigned char* run1 = run0 + RUN;
            unsigned pa[G], pb[G], steps0[G], steps1[G];
            load_pairs(run0 + 128 * G + c * 4 * G, pa);
            load_pairs(run0 + 128 * G + (c + 4) * 4 * G, pb);
#pragma unroll
            for (int g = 0; g < G; ++g) steps0[g] = __byte_perm(pa[g], pb[g], 0x5410);
            load_pairs(run1 + 128 * G + c * 4 * G, pa);
            load_pairs(run1 + 128 * G + (c + 4) * 4 * G, pb);
#pragma unroll
            for (int g = 0; g < G; ++g) steps1[g] = __byte_perm(pa[g], pb[g], 0x5410);
            // row g of the side sums: m of group r (rows beyond the groups repeat them and are not looked at)
            const unsigned* at0 = reinterpret_cast<const unsigned*>(run0 + 128 * G + 4 * (r % G));
            const unsigned* at1 = reinterpret_cast<const unsigned*>(run1 + 128 * G + 4 * (r % G));
            const unsigned base0 = __byte_perm(at0[c * G], at0[(c + 4) * G], 0x7632), base1 = __byte_perm(at1[c * G], at1[(c + 4) * G], 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if constexpr (TWICE) {
                    mma(side[nt], base0, one, base1, one, times_bf16(second ? rest[u][nt][0] : p[u][nt][0], sink), times_bf16(second ? rest[u][nt][1] : p[u][nt][1], sink));
                    rest[u][nt][0] &= second;
                    rest[u][nt][1] &= second;
                } else {
                    mma(side[nt], base0, one, base1, one, times_bf16(p[u][nt][0], sink), times_bf16(p[u][nt][1], sink));
                    mma(side[nt], base0, one, base1, one, times_bf16(rest[u][nt][0], sink), times_bf16(rest[u][nt][1], sink));
                }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const unsigned char* from0 = run0 + g * 128 + (r >> 1) * 4;
                const unsigned char* from1 = run1 + g * 128 + (r >> 1) * 4;
                const unsigned x = __byte_perm(*reinterpret_cast<const unsigned*>(from0 + c * 16), *reinterpret_cast<const unsigned*>(from0 + (c + 4) * 16), half);
                const unsigned y = __byte_perm(*reinterpret_cast<const unsigned*>(from1 + c * 16), *reinterpret_cast<const unsigned*>(from1 + (c + 4) * 16), half);
                const unsigned xs = x >> 8, ys = y >> 8;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    // p s, what that rounds off (a number of 8 bits) and the rest's product; TWICE: 0 and 0 in the first columns, which gives p s again
                    const unsigned ps0 = times_bf16(p[u][nt][0], steps0[g]), ps1 = times_bf16(p[u][nt][1], steps1[g]);
                    const unsigned less0 = TWICE ? minus_bf16(ps0) & second : minus_bf16(ps0), less1 = TWICE ? minus_bf16(ps1) & second : minus_bf16(ps1);
                    const unsigned off0 = fma_bf16(rest[u][nt][0], steps0[g], fma_bf16(p[u][nt][0], steps0[g], less0));
                    const unsigned off1 = fma_bf16(rest[u][nt][1], steps1[g], fma_bf16(p[u][nt][1], steps1[g], less1));
                    if constexpr (!TWICE) {
                        mma(acc[nt][g][0], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, ps0, ps1);
                        mma(acc[nt][g][1], xs & 0x000f000fu, xs & 0x00f000f0u, ys & 0x000f000fu, ys & 0x00f000f0u, ps0, ps1);
                    }
                    mma(acc[nt][g][0], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, off0, off1);
                    mma(acc[nt][g][1], xs & 0x000f000fu, xs & 0x00f000f0u, ys & 0x000f000fu, ys & 0x00f000f0u, off0, off1);
                }
            }
        }
        __syncwarp();
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    copies_wait<0>();

    // ---- the block's rows: [WARPS][8 rows][D] floats at a time
    const bool alone = span.count == 1;
    float* rows_o = reinterpret_cast<float*>(shared);
    const float down = scalbnf(1.f, 33 - (int)lift);
    if constexpr (TWICE) {                       // the second columns
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            side[0][i] += __shfl_xor_sync(0xffffffffu, side[0][i], 2);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                acc[0][g][0][i] += __shfl_xor_sync(0xffffffffu, acc[0][g][0][i], 2);
                acc[0][g][1][i] += __shfl_xor_sync(0xffffffffu, acc[0][g][1][i], 2);
            }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if (r == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                row_ml[warp][nt * 8 + 2 * c + i][0] = most[nt][i] == NOTHING ? -INFINITY : most[nt][i] * unit[nt][i];
                row_ml[warp][nt * 8 + 2 * c + i][1] = side[nt][2 + i];
            }
        }
        __syncthreads();               // the ring, or the rows before these, are done with
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float bases = __shfl_sync(0xffffffffu, side[nt][i], 4 * g + c);
                const float add = (marked[nt][i] >> g & 1) ? __int_as_float(0x7fc00000) : bases;
                float4 o;                                  // 2^133 2^-lift is beyond float32 for a lift below 6: in two steps
                o.x = fmaf(acc[nt][g][0][i] * 0x1p100f, down, add);
                o.y = fmaf(acc[nt][g][0][2 + i] * 0x1p96f, down, add);
                o.z = fmaf(acc[nt][g][1][i] * 0x1p100f, down, add);
                o.w = fmaf(acc[nt][g][1][2 + i] * 0x1p96f, down, add);
                *reinterpret_cast<float4*>(rows_o + (warp * 8 + 2 * c + i) * D + g * KV4_GROUP + 4 * r) = o;
            }
        __syncthreads();
        for (int i = threadIdx.x; i < (TWICE ? 4 : 8) * (D / 4); i += 32 * WARPS) {
            const int of = i / (D / 4), d = i % (D / 4) * 4, row = row0 + nt * 8 + of;
            if (row >= all_rows) break;
            float peak = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) peak = fmaxf(peak, row_ml[w][nt * 8 + of][0]);
            const float against = peak == -INFINITY ? 0.f : peak;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float keep = fast_exp2(row_ml[w][nt * 8 + of][0] - against);
                const float4 o = *reinterpret_cast<const float4*>(rows_o + (w * 8 + of) * D + d);
                sum.x = fmaf(o.x, keep, sum.x); sum.y = fmaf(o.y, keep, sum.y);
                sum.z = fmaf(o.z, keep, sum.z); sum.w = fmaf(o.w, keep, sum.w);
                l = fmaf(row_ml[w][nt * 8 + of][1], keep, l);
            }
            const int head = kv * share + row % share;
            if (alone) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                *reinterpret_cast<uint2*>(a.out + ((size_t)(first_token + row / share) * a.q_heads + head) * D + d)
                    = make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv));
            } else if (a.clustered) {
                *reinterpret_cast<float4*>(rows_o + (WARPS * 8 + nt * 8 + of) * D + d) = sum;
                if (d == 0) joint_ml[nt * 8 + of] = make_float2(peak, l);
            } else {
                const size_t slot = ((size_t)(more.x + row / share) * a.q_heads + head) * a.n_spans + my_span;
                *reinterpret_cast<float4*>(a.part_o + slot * D + d) = sum;
                if (d == 0) *reinterpret_cast<float2*>(a.part_ml + slot * 2) = make_float2(peak, l);
            }
        }
    }
    if (alone) return;
    if (a.clustered) {
        // ---- every block joins a part of the rows, out of the shared memory of all
        cluster_sync_all();
        const unsigned mine_o = (unsigned)__cvta_generic_to_shared(rows_o + WARPS * 8 * D), mine_ml = (unsigned)__cvta_generic_to_shared(joint_ml);
        for (int i = my_span * 32 * WARPS + threadIdx.x; i < rows * (D / 4); i += span.count * 32 * WARPS) {
            const int of = i / (D / 4), d = i % (D / 4) * 4, row = row0 + of, head = kv * share + row % share;
            float peak = -INFINITY, l = 0.f;
            for (int s = 0; s < span.count; ++s) peak = fmaxf(peak, cluster_load(mine_ml + of * 8, s));
            const float against = peak == -INFINITY ? 0.f : peak;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int s = 0; s < span.count; ++s) {
                const float2 ml = cluster_load2(mine_ml + of * 8, s);
                const float4 o = cluster_load4(mine_o + (of * D + d) * 4, s);
                const float keep = fast_exp2(ml.x - against);
                sum.x = fmaf(o.x, keep, sum.x); sum.y = fmaf(o.y, keep, sum.y);
                sum.z = fmaf(o.z, keep, sum.z); sum.w = fmaf(o.w, keep, sum.w);
                l = fmaf(ml.y, keep, l);
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            *reinterpret_cast<uint2*>(a.out + ((size_t)(first_token + row / share) * a.q_heads + head) * D + d)
                = make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv));
        }
        cluster_sync_all();                  // the others' reads are done
        return;
    }
    // ---- the last block of these rows joins the spans
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        int* ticket = a.tickets + (size_t)more.x * a.q_heads + kv * all_rows + row0 / ROWS;
        last_block = atomicAdd(ticket, 1) == span.count - 1;
        if (last_block) *ticket = 0;
    }
    __syncthreads();
    if (!last_block) return;
    __threadfence();
    float* weight = reinterpret_cast<float*>(shared);          // [8 NT][n_spans], then the sums of the rows
    for (int of = warp; of < rows; of += WARPS) {
        const int row = row0 + of;
        const size_t slot = ((size_t)(more.x + row / share) * a.q_heads + kv * share + row % share) * a.n_spans;
        float peak = -INFINITY, l = 0.f;
        for (int s = lane; s < span.count; s += 32) peak = fmaxf(peak, __ldcg(a.part_ml + (slot + s) * 2));
        peak = warp_max(peak);
        const float against = peak == -INFINITY ? 0.f : peak;
        for (int s = lane; s < span.count; s += 32) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.part_ml + (slot + s) * 2));
            const float keep = fast_exp2(ml.x - against);
            weight[of * a.n_spans + s] = keep;
            l = fmaf(ml.y, keep, l);
        }
        l = warp_sum(l);
        if (lane == 0) row_ml[0][of][0] = l == 0.f ? 0.f : 1.f / l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (D / 4); i += 32 * WARPS) {
        const int of = i / (D / 4), d = i % (D / 4) * 4, row = row0 + of, head = kv * share + row % share;
        const float* from = a.part_o + ((size_t)(more.x + row / share) * a.q_heads + head) * a.n_spans * D + d;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int s = 0; s < span.count; ++s) {
            const float4 o = __ldcg(reinterpret_cast<const float4*>(from + (size_t)s * D));
            const float keep = weight[of * a.n_spans + s];
            sum.x = fmaf(o.x, keep, sum.x); sum.y = fmaf(o.y, keep, sum.y);
            sum.z = fmaf(o.z, keep, sum.z); sum.w = fmaf(o.w, keep, sum.w);
        }
        const float inv = row_ml[0][of][0];
        *reinterpret_cast<uint2*>(a.out + ((size_t)(first_token + row / share) * a.q_heads + head) * D + d)
            = make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv));
    }
}

template <int NT, bool TWICE>
static int launch(const Kv4Few& a, int n, int most_rows, cudaStream_t stream) {
    const int ring = WARPS * STAGES * STAGE_BYTES, rows = WARPS * 8 * D * 4, weights = 8 * NT * a.n_spans * 4;
    const int smem = ring > rows ? (ring > weights ? ring : weights) : (rows > weights ? rows : weights);
    static QilPerDevice configured;
    const cudaError_t reserved = configured.once(qil_device(), [] {
        const cudaError_t e = cudaFuncSetAttribute(kv4_few_kernel<NT, TWICE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
        return e != cudaSuccess ? e : cudaFuncSetAttribute(kv4_few_kernel<NT, TWICE>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    if (reserved != cudaSuccess) QIL_REFUSE("kv4: cannot reserve shared memory or clusters of %d blocks: %s", MOST_CLUSTER, cudaGetErrorString(reserved));
    constexpr int ROWS = TWICE ? 4 : 8 * NT;
    const dim3 grid(a.n_spans * ((most_rows + ROWS - 1) / ROWS), a.kv_heads, n);
    if (grid.y > 65535 || grid.z > 65535) QIL_REFUSE("kv4: %d segments of %d kv heads", n, a.kv_heads);
    const cudaError_t e = a.clustered ? qil_launch_clusters(kv4_few_kernel<NT, TWICE>, grid, dim3(32 * WARPS), smem, a.n_spans, stream, a)
                                      : qil_launch_chained(kv4_few_kernel<NT, TWICE>, grid, dim3(32 * WARPS), smem, stream, a);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        snprintf(qil_error_text, sizeof(qil_error_text), "%s", cudaGetErrorString(e));
        return (int)e;
    }
    return 0;
}

extern "C" int qil_kv4_few_head_dim() { return D; }
extern "C" int qil_kv4_few_most_spans() { return MOST_SPANS; }
extern "C" int qil_kv4_few_blocks_a_sm(int nt) { return blocks_a_sm(nt); }

// info: see Kv4Few; most_tokens: segments of more are left alone; nt: 8-row tiles a block takes, 1 or 2.
struct Kv4FewCall {
    const void *q, *pages;
    void* out;
    const void* info;
    void *part_o, *part_ml, *tickets;
    const void* block_table;
    cudaStream_t stream;
    float scale;
    int n, most_tokens, nt, n_spans, table_height, table_width, q_heads, kv_heads, page_size, num_pages, window, clustered, settled;
};
extern "C" int qil_kv4_few_call_bytes() { return sizeof(Kv4FewCall); }
extern "C" int qil_kv4_few(const void* packed) {
    const auto [q, pages, out, info, part_o, part_ml, tickets, block_table, stream, scale, n, most_tokens, nt, n_spans, table_height, table_width,
                q_heads, kv_heads, page_size, num_pages, window, clustered, settled] = kv4_call<Kv4FewCall>(packed);
    if (n <= 0) return 0;
    if (page_size <= 0 || page_size % 8) QIL_REFUSE("pages of a multiple of 8 positions, not %d", page_size);
    if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || n_spans < 1 || n_spans > (clustered ? MOST_CLUSTER : MOST_SPANS) || most_tokens < 1 || window < 0)
        QIL_REFUSE("%d query heads, %d kv heads, %d spans", q_heads, kv_heads, n_spans);
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)pages | (uintptr_t)info | (uintptr_t)part_o) & 15) QIL_REFUSE("kv4: operands must be 16-byte aligned");
    const Kv4Few a = {(const bf16*)q, (const uint8_t*)pages, (bf16*)out, (const int*)info, (float*)part_o, (float*)part_ml, (int*)tickets,
                      {(const int*)block_table, table_height, table_width, page_size, num_pages}, n_spans, q_heads, kv_heads, window, most_tokens, clustered,
                      settled,
                      scale * 1.4426950408889634f};
    const int rows = most_tokens * (q_heads / kv_heads);
    if (nt == 1) return rows <= 4 ? launch<1, true>(a, n, rows, stream) : launch<1, false>(a, n, rows, stream);
    if (nt == 2) return launch<2, false>(a, n, rows, stream);
    QIL_REFUSE("kv4: %d tiles of rows a block", nt);
}
