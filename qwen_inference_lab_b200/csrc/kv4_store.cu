// Rows into pages of 4 bits and back (layout and rounding: kv4.h).
//
// kv4_store: the tail of a q/k/v projection.  Per head r = 1 / sqrt(mean x^2 + eps), y = x r w (norm), then the first rot_dims
// dimensions turn by the position's angles, (u, v) -> (u c - v s, v c + u s), with u, v half of the rotated dimensions apart or
// neighbours; c, s come from a float32 table or from frequencies (angle = position * frequency in 64 bits: in 32 a position
// beyond 2^17 loses 0.01 rad).  Without weights the norm may come after the turn ("unit heads").  Queries are rounded once to
// their type and written; keys and values are cut into groups and coded.  Keys are computed in 64 bits: which code an element
// gets is a step function of its value, and so is the same here as in any other arithmetic that keeps 64 bits, where in 32 bits one of
// 10^5 elements would land on the other side of a border.  Queries have no borders and stay in 32 bits.
//
// 64-bit arithmetic is what such a kernel would take its time for, and hardly any element needs it: a row is computed in 32 bits first,
// with a bound on what that may be off (up to 15 roundings of the two products that a turn adds), and again in 64 bits only if a step, a
// base or a code could come out otherwise within that bound (a row or two in a hundred).  Such a row keeps its warp waiting for 3.9 us, and
// among 64 tokens there is one nearly always: 64 tokens of 32 + 2 x 8 heads of 128 take 6.8 us, 3.6 if none had to; 2048 take 26.5 and 22.9.
// (The same in pairs of 32-bit numbers with an exact sum and product waits 2.9: not worth a third way.)  The rest is instructions: a lane takes 8
// neighbouring elements, so that a head of 128 is half a warp and a group's codes are one word of each of four lanes, and a token's
// cosines and sines times the weights stay in registers from head to head: (x r w) c -+ (x' r w') s is r (x (w c) -+ x' (w' s)).
//
// kv4_spread: the rows of a prompt portion's context for the kernel that attends to 16-bit operands (attention_tc.cu with float16 keys):
// float16 keys and values with a power of two taken out of each per page of 64 and head; where a group of values is NaN, zeros and a mark.
// An element is off by 2^-11 of itself where it is not smaller than 2^-23 of the largest of its page and head, by 2^-33 of that largest below.
//
// kv4_read: rows of requests as ordinary pages [page][2][kv head][slot][d] of float32 or bfloat16.
#include "kv4.h"
#include <cuda_fp16.h>

QIL_ERROR_STORAGE

// Warps a block, blocks an SM.  Measured (us, 64 / 256 / 2048 tokens): 8 x 4 7.2 / 9.3 / 31.5, 4 x 6 6.5 / 8.2 / 31.0, 4 x 7 6.7 / 8.8 / 26.9, 4 x 8 7.0 /
// 9.5 / 26.7, 2 x 14 7.2 / 9.8 / 26.1.
static constexpr int STORE_WARPS = 4, STORE_BLOCKS = 7;

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
    Kv4Table table_of;
    int tokens, q_heads, kv_heads, dim;
    int vectors;                    // four elements are read and written at a time: columns, strides and pointers allow it
};

__device__ __forceinline__ float shfl_xor(float v, int mask) { return __shfl_xor_sync(0xffffffffu, v, mask); }
__device__ __forceinline__ double shfl_xor(double v, int mask) { return __shfl_xor_sync(0xffffffffu, v, mask); }
__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
// Smallest and largest of a group, in its four lanes.
template <typename R> __device__ __forceinline__ void range_of(const R (&y)[8], R& lo, R& hi) {
    lo = smaller(smaller(smaller(y[0], y[1]), smaller(y[2], y[3])), smaller(smaller(y[4], y[5]), smaller(y[6], y[7])));
    hi = larger(larger(larger(y[0], y[1]), larger(y[2], y[3])), larger(larger(y[4], y[5]), larger(y[6], y[7])));
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = smaller(lo, shfl_xor(lo, o));
        hi = larger(hi, shfl_xor(hi, o));
    }
}
__device__ __forceinline__ unsigned pair_of(bf16 step, bf16 base) {
    return (unsigned)__bfloat16_as_ushort(base) << 16 | __bfloat16_as_ushort(step);
}
static constexpr unsigned NAN_PAIR = 0x7fc07fc0u;

// Eight elements a lane, exact: the definition.  A code is the quotient's nearest whole number without a division: a step has 8
// bits, so the products with it are exact, and 32 bits are enough to be next to it.
__device__ __forceinline__ void code_exact(const double (&y)[8], unsigned& codes, unsigned& pair) {
    double lo, hi;
    range_of(y, lo, hi);
    bool good = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) good = good && isfinite(y[i]);
    good = ((__ballot_sync(0xffffffffu, good) >> (threadIdx.x & 28)) & 0xfu) == 0xfu;          // in all lanes of the group
    const bf16 base = __float2bfloat16_rn(__double2float_rn(lo));
    const bf16 step = __float2bfloat16_rn(__double2float_rn((hi - lo) / 15.0));
    const double m = (double)__bfloat162float(base), s = (double)__bfloat162float(step);
    good = good && isfinite(m) && isfinite(s);
    codes = 0;
    if (good && s > 0.0) {
        const double middling = s < 0x1p-64 ? 0x1p80 : s > 0x1p64 ? 0x1p-80 : 1.0;           // where steps and distances are ordinary floats
        const float inverse = 1.f / (float)(s * middling);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double d = y[i] - m;
            int n = min(max(__float2int_rn((float)(d * middling) * inverse), 0), 15);
            const double above = fma(-((double)n + 0.5), s, d), below = fma(-((double)n - 0.5), s, d);
            n += above > 0.0 || (above == 0.0 && (n & 1)) ? 1 : below < 0.0 || (below == 0.0 && (n & 1)) ? -1 : 0;
            codes |= (unsigned)min(max(n, 0), 15) << (4 * i);
        }
    }
    pair = good ? pair_of(step, base) : NAN_PAIR;
}
// The same from elements of which those of this lane's group are off by `off` at most; false where that could make a difference.
// Elements that are exact (EXACT, off = 0) as their distances from the base are, as bfloat16 values are, lie between two codes often
// (s times a half is a number like they are): the sign of (y - m) - (n + 1/2) s, one rounding, decides them, and 0 is a tie.
template <bool EXACT> __device__ __forceinline__ bool code_within(const float (&y)[8], float off, unsigned& codes, unsigned& pair) {
    float lo, hi;
    range_of(y, lo, hi);
    const float range = hi - lo, wide = fmaf(range, 2.4e-7f, 2.f * off) * 1.001f;      // what the range may be off, its own rounding included
    const bf16 base = __float2bfloat16_rn(lo - off), step = __float2bfloat16_rn((range - wide) * ((1.f / 15.f) * (1.f - 2.4e-7f)));
    const bf16 base_up = __float2bfloat16_rn(lo + off), step_up = __float2bfloat16_rn((range + wide) * ((1.f / 15.f) * (1.f + 2.4e-7f)));
    const float m = __bfloat162float(base), s = __bfloat162float(step);
    bool sure = pair_of(step, base) == pair_of(step_up, base_up) && s > 1e-30f && hi < 1e30f && lo > -1e30f;
    const float inverse = 1.f / s, most = 0.5f - fmaf(off, inverse, 8e-6f);            // 16 codes' three roundings are 3e-6
    codes = 0;
    float furthest = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = (y[i] - m) * inverse;
        const float up = fminf(fmaxf(t, 0.f), 15.f) + 12582912.f;                      // 1.5 2^23: its last bits are the whole number, ties to even
        furthest = fmaxf(furthest, fabsf(t - (up - 12582912.f)));
        sum += t;                                                                      // NaN stays in a sum, not in a maximum
        codes |= (__float_as_uint(up) & 15u) << (4 * i);
    }
    pair = pair_of(step, base);
    sure = sure && sum == sum;
    if (EXACT && sure && !(furthest < most)) {
        codes = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = y[i] - m, below = floorf(fminf(fmaxf(d * inverse, 0.f), 15.f));
            const float side = fmaf(-(below + 0.5f), s, d);
            const unsigned n = (unsigned)(int)below;
            sure = sure && d + m == y[i] && y[i] - d == m;
            codes |= min(n + (side > 0.f || (side == 0.f && (n & 1u)) ? 1u : 0u), 15u) << (4 * i);
        }
        return sure;
    }
    return sure && furthest < most;
}

// Eight elements of a row as they lie there, and as floats.
struct EightBf16 {
    uint4 v;
    __device__ __forceinline__ void load(const bf16* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void one_by_one(const bf16* p) {
        const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
        v = make_uint4(u[0] | (unsigned)u[1] << 16, u[2] | (unsigned)u[3] << 16, u[4] | (unsigned)u[5] << 16, u[6] | (unsigned)u[7] << 16);
    }
    __device__ __forceinline__ void zero() { v = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ EightBf16 of_lane(int lane) const {
        EightBf16 o;
        o.v = make_uint4(__shfl_sync(0xffffffffu, v.x, lane), __shfl_sync(0xffffffffu, v.y, lane), __shfl_sync(0xffffffffu, v.z, lane), __shfl_sync(0xffffffffu, v.w, lane));
        return o;
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};
struct EightF32 {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = reinterpret_cast<const float4*>(p)[0];
        b = reinterpret_cast<const float4*>(p)[1];
    }
    __device__ __forceinline__ void one_by_one(const float* p) {
        a = make_float4(p[0], p[1], p[2], p[3]);
        b = make_float4(p[4], p[5], p[6], p[7]);
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ EightF32 of_lane(int lane) const {
        EightF32 o;
        o.a = make_float4(__shfl_sync(0xffffffffu, a.x, lane), __shfl_sync(0xffffffffu, a.y, lane), __shfl_sync(0xffffffffu, a.z, lane), __shfl_sync(0xffffffffu, a.w, lane));
        o.b = make_float4(__shfl_sync(0xffffffffu, b.x, lane), __shfl_sync(0xffffffffu, b.y, lane), __shfl_sync(0xffffffffu, b.z, lane), __shfl_sync(0xffffffffu, b.w, lane));
        return o;
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
};
template <typename T> struct Eight;
template <> struct Eight<bf16> { typedef EightBf16 type; };
template <> struct Eight<float> { typedef EightF32 type; };

__device__ __forceinline__ unsigned two_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(bf16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(two_bf16(v[0], v[1]), two_bf16(v[2], v[3]), two_bf16(v[4], v[5]), two_bf16(v[6], v[7]));
}

// 1 / sqrt(v): queries have no borders and can do with 2^-22.
__device__ __forceinline__ float root_of(float v, bool near) { return near ? rsqrtf(v) : 1.f / sqrtf(v); }
// Sum over the lanes of a head.
template <int LANES, typename R> __device__ __forceinline__ R head_sum(R v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += shfl_xor(v, o);
    return v;
}

// Where an element's angle comes from: element d < rot_dims belongs to pair pair_of(d); its partner is other_of(d), and it is the second
// of the two where second(d).
struct Turn {
    int rot_dims, half, interleaved;
    __device__ __forceinline__ int other_of(int d) const { return d >= rot_dims ? d : interleaved ? d ^ 1 : d < half ? d + half : d - half; }
    __device__ __forceinline__ int pair_at(int d) const { return interleaved ? d >> 1 : d < half ? d : d - half; }
    __device__ __forceinline__ bool second(int d) const { return interleaved ? (d & 1) != 0 : d >= half; }
};
// Cosine and sine of a pair at a position, gain included.
__device__ __forceinline__ void angle_of(const Kv4Store& a, int pos, int pair, double& c, double& s) {
    if (a.table != nullptr) {
        const float* row = a.table + (size_t)min(max(pos, 0), a.table_rows - 1) * a.rot_dims;
        c = row[pair];
        s = row[(a.rot_dims >> 1) + pair];
    } else {
        sincos((double)pos * (double)a.freq[pair], &s, &c);
        c *= (double)a.gain;
        s *= (double)a.gain;
    }
}
// A warp's keys in 64 bits, and their codes.  Out of line: few rows come here, and its registers are twice the others'.  All that it needs
// comes by value, in registers: read through a pointer to the kernel's arguments it is in no cache.
template <typename W, int LANES>
__device__ __noinline__ uint2 keys_exact(const W* weight, const double2* angles, float eps, int norm, int dim, int rot_dims, int interleaved, int d0,
                                         float4 x0, float4 x1, float4 v0, float4 v1) {
    const Turn turn = {rot_dims, rot_dims >> 1, interleaved};
    const float own[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w}, partner[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    double exact[8], r = 1.0, sq = 0.0;
    if (norm == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += (double)own[i] * (double)own[i];
        r = rsqrt(head_sum<LANES>(sq) / (double)dim + (double)eps);
        sq = 0.0;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        double u = (double)own[i], v = (double)partner[i];
        if (norm == 1 && d < dim) {
            u = u * r * (double)to_f32<W>(weight[d]);
            v = v * r * (double)to_f32<W>(weight[turn.other_of(d)]);
        }
        if (d < rot_dims) {
            const double2 at = angles[turn.pair_at(d)];
            u = turn.second(d) ? u * at.x + v * at.y : u * at.x - v * at.y;
        }
        exact[i] = u;
        sq += u * u;
    }
    if (norm == 2) {
        r = rsqrt(head_sum<LANES>(sq) / (double)dim + (double)eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) exact[i] *= r;
    }
    uint2 found;
    code_exact(exact, found.x, found.y);
    return found;
}
__device__ __noinline__ uint2 values_exact(float4 x0, float4 x1) {
    const double exact[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
    uint2 found;
    code_exact(exact, found.x, found.y);
    return found;
}

// A block: a token and every (gridDim.y)th set of STORE_WARPS steps, from the last on; a warp takes 32 / LANES heads of one kind a step, LANES lanes of 8
// elements each (the first dim / 8 of them; a power of two).
template <int KIND> struct Kind { static constexpr int kind = KIND; };
template <typename T, typename W, int LANES>
__global__ void __launch_bounds__(32 * STORE_WARPS, STORE_BLOCKS) kv4_store_kernel(const __grid_constant__ Kv4Store a) {
    constexpr int HEADS = 32 / LANES;
    // what an element and its partner are multiplied by: cosines times own weights, signed sines times partners', of queries and of keys
    __shared__ __align__(16) float factor[2][2][8 * LANES];
    __shared__ double2 angles[4 * LANES];                  // cosine and sine of the pairs
    qil_wait_for_producer();
    qil_release_consumer();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, token = blockIdx.x;
    const int pos = a.positions[token], half = a.rot_dims >> 1, groups = a.dim / KV4_GROUP;
    const Turn turn = {a.rot_dims, half, a.interleaved};
    int page = -1;
    if (a.kv_heads) page = a.table_of.page(a.token_row[token], pos);
    for (int d = threadIdx.x; d < 8 * LANES; d += 32 * STORE_WARPS) {
        double cosine = 1.0, sine = 0.0;
        if (d < a.rot_dims) {
            angle_of(a, pos, turn.pair_at(d), cosine, sine);
            if (!turn.second(d)) angles[turn.pair_at(d)] = make_double2(cosine, sine);
        }
        const float c = (float)cosine, s = turn.second(d) ? (float)sine : -(float)sine;
        const bool weighs = a.norm == 1 && d < a.dim;
        const W* q_weight = reinterpret_cast<const W*>(a.q_weight);
        const W* k_weight = reinterpret_cast<const W*>(a.k_weight);
        factor[0][0][d] = weighs ? c * to_f32<W>(q_weight[d]) : c;
        factor[0][1][d] = weighs ? s * to_f32<W>(q_weight[turn.other_of(d)]) : s;
        factor[1][0][d] = weighs ? c * to_f32<W>(k_weight[d]) : c;
        factor[1][1][d] = weighs ? s * to_f32<W>(k_weight[turn.other_of(d)]) : s;
    }
    __syncthreads();
    const int sub = lane / LANES, l = lane % LANES, d0 = 8 * l;
    const int steps_q = (a.q_heads + HEADS - 1) / HEADS, steps_kv = (a.kv_heads + HEADS - 1) / HEADS;
    // where a halves layout's other elements lie: whole lanes away, or anywhere
    const bool by_lanes = half % 8 == 0;
    const int other_lane = lane + (d0 >= a.rot_dims ? 0 : d0 < half ? half / 8 : -(half / 8));
    const int slot = pos % a.table_of.page_size;
    const int head_bytes = (a.table_of.page_size >> 3) * kv4_run_bytes(groups);
    uint8_t* const to = page < 0 ? nullptr : a.pages + kv4_run_at(page, 0, 0, slot, a.kv_heads, a.table_of.page_size, groups);
    const int code_at = kv4_code_at(l >> 2, slot) + (l & 3) * 4, pair_at = kv4_pair_at(l >> 2, slot, groups);
    float cw[8], sw[8];
    auto load_factors = [&](int kind) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 c = *reinterpret_cast<const float4*>(&factor[kind][0][d0 + i]), s = *reinterpret_cast<const float4*>(&factor[kind][1][d0 + i]);
            cw[i] = c.x; cw[i + 1] = c.y; cw[i + 2] = c.z; cw[i + 3] = c.w;
            sw[i] = s.x; sw[i + 1] = s.y; sw[i + 2] = s.z; sw[i + 3] = s.w;
        }
    };
    // the `index`th set of heads of a kind: queries, keys, values
    auto step = [&](auto of, int index) {
        constexpr int now = decltype(of)::kind;
        const int head = index * HEADS + sub;
        const bool mine = head < (now == 0 ? a.q_heads : a.kv_heads) && d0 < a.dim;
        const T* src = reinterpret_cast<const T*>(a.proj) + (size_t)token * a.ld + (now == 0 ? a.q_col : now == 1 ? a.k_col : a.v_col) + head * a.dim;
        typename Eight<T>::type own, partner;
        own.zero();
        if (mine) {
            if (a.vectors) own.load(src + d0);
            else own.one_by_one(src + d0);
        }
        float x[8], y[8], xp[8], off = 0.f;
        own.floats(x);
        if constexpr (now < 2) {
            if (a.interleaved) {
#pragma unroll
                for (int i = 0; i < 8; ++i) xp[i] = x[i ^ 1];
            } else if (by_lanes) {
                partner = own.of_lane(other_lane & 31);
                partner.floats(xp);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) xp[i] = mine ? to_f32<T>(src[turn.other_of(d0 + i)]) : 0.f;
            }
            if (a.rot_dims < a.dim) {              // what is not turned has nothing to add: not an infinity times a sine of zero either
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (d0 + i >= a.rot_dims) xp[i] = 0.f;
            }
            float r = 1.f;
            if (a.norm == 1) {
                float sq = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) sq = fmaf(x[i], x[i], sq);
                r = root_of(head_sum<LANES>(sq) / (float)a.dim + a.eps, now == 0);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float turned = xp[i] * sw[i];
                y[i] = fmaf(x[i], cw[i], turned);
                if (now == 1) off = fmaxf(off, fmaf(fabsf(x[i]), fabsf(cw[i]), fabsf(turned)));
            }
            if (a.norm == 2) {
                float sq = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) sq = fmaf(y[i], y[i], sq);
                r = root_of(head_sum<LANES>(sq) / (float)a.dim + a.eps, now == 0);
            }
            if (a.norm) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] *= r;
                off *= r < 1e13f ? r : INFINITY;                                             // squares of less than 1e-26 lose bits
            }
        }
        if constexpr (now == 0) {
            if (mine) store8(reinterpret_cast<T*>(a.q_out) + ((size_t)token * a.q_heads + head) * a.dim + d0, y);
        } else {
            unsigned codes, pair;
            bool sure;
            if constexpr (now == 1) {
                // 15 roundings of the two products; where the norm is of the turned head their errors go into its sum of squares, and so
                // from any element into any other: up to 60 roundings of the largest (one large element among 255 equal ones)
#pragma unroll
                for (int o = 1; o < LANES; o <<= 1)
                    if (o < 4 || a.norm == 2) off = fmaxf(off, __shfl_xor_sync(0xffffffffu, off, o));
                sure = code_within<false>(y, off * (a.norm == 2 ? 0x1p-18f : 0x1p-20f), codes, pair);
            } else {
                sure = code_within<true>(x, 0.f, codes, pair);
            }
            if (__any_sync(0xffffffffu, mine && !sure)) {
                const float4 x0 = make_float4(x[0], x[1], x[2], x[3]), x1 = make_float4(x[4], x[5], x[6], x[7]);
                uint2 found;
                if constexpr (now == 1)
                    found = keys_exact<W, LANES>(reinterpret_cast<const W*>(a.k_weight), angles, a.eps, a.norm, a.dim, a.rot_dims, a.interleaved, d0, x0, x1,
                                                 make_float4(xp[0], xp[1], xp[2], xp[3]), make_float4(xp[4], xp[5], xp[6], xp[7]));
                else found = values_exact(x0, x1);
                codes = found.x;
                pair = found.y;
            }
            if (mine) {
                uint8_t* run = to + (size_t)((now - 1) * a.kv_heads + head) * head_bytes;
                *reinterpret_cast<unsigned*>(run + code_at) = codes;
                if ((l & 3) == 0) *reinterpret_cast<unsigned*>(run + pair_at) = pair;
            }
        }
    };
    // Every warp takes values or keys, which take longest, and then queries; a loop of its own a kind (one for all of them, with branches inside,
    // took 30.7 us of 2048 tokens instead of 26.9).
    const int stride = gridDim.y * STORE_WARPS;
    int at = blockIdx.y * STORE_WARPS + warp;
    for (; at < steps_kv; at += stride)
        if (page >= 0) step(Kind<2>(), at);
    at -= steps_kv;
    if (at < steps_kv) load_factors(1);
    for (; at < steps_kv; at += stride)
        if (page >= 0) step(Kind<1>(), at);
    at -= steps_kv;
    load_factors(0);
    for (; at < steps_q; at += stride) step(Kind<0>(), at);
}

struct Kv4StoreCall {
    const void* proj;
    long long ld;
    void *q_out, *pages;
    const void *q_weight, *k_weight, *table, *freq, *positions, *token_row, *block_table;
    cudaStream_t stream;
    float eps, gain;
    int q_col, k_col, v_col, norm, table_rows, rot_dims, interleaved, table_height, table_width, tokens, q_heads, kv_heads, dim, page_size, num_pages,
        act, weight;
};
extern "C" int qil_kv4_store(const void* packed) {
    const auto [proj, ld, q_out, pages, q_weight, k_weight, table, freq, positions, token_row, block_table, stream, eps, gain, q_col, k_col, v_col,
                norm, table_rows, rot_dims, interleaved, table_height, table_width, tokens, q_heads, kv_heads, dim, page_size, num_pages, act,
                weight] = kv4_call<Kv4StoreCall>(packed);
    if (tokens <= 0) return 0;
    if (dim <= 0 || dim > KV4_MAX_DIM || dim % KV4_GROUP) QIL_REFUSE("head sizes 32, 64, ..., %d, not %d", KV4_MAX_DIM, dim);
    if (page_size <= 0 || page_size % 8) QIL_REFUSE("pages of a multiple of 8 positions, not %d", page_size);
    if (rot_dims < 0 || rot_dims > dim || rot_dims % 2 || (rot_dims && table == nullptr && freq == nullptr)
        || (table != nullptr && table_rows <= 0))
        QIL_REFUSE("%d rotated dimensions of %d", rot_dims, dim);
    if (q_heads < 0 || kv_heads < 0 || q_heads + kv_heads == 0) QIL_REFUSE("no heads");
    Kv4Store a = {proj, ld, q_col, k_col, v_col, q_out, (uint8_t*)pages, q_weight, k_weight, eps, norm, (const float*)table, table_rows,
                  (const float*)freq, gain, rot_dims, interleaved, (const int*)positions, (const int*)token_row,
                  {(const int*)block_table, table_height, table_width, page_size, num_pages}, tokens, q_heads, kv_heads, dim, 0};
    const int eight = act == QIL_BF16 ? 8 : 4;               // elements of 16 bytes
    a.vectors = ld % eight == 0 && q_col % eight == 0 && k_col % eight == 0 && v_col % eight == 0 && (uintptr_t)proj % 16 == 0;
    if ((uintptr_t)q_out % 16) QIL_REFUSE("queries out must start on a 16-byte boundary");
    const int lanes = dim <= 32 ? 4 : dim <= 64 ? 8 : dim <= 128 ? 16 : 32, heads = 32 / lanes;
    const int steps = (q_heads + heads - 1) / heads + 2 * ((kv_heads + heads - 1) / heads), sets = (steps + STORE_WARPS - 1) / STORE_WARPS;
    // as many blocks a token as fill the GPU once, a step a warp at most
    const int fit = 148 * STORE_BLOCKS / tokens;              // 148 SMs
    const dim3 grid(tokens, fit < 1 ? 1 : fit < sets ? fit : sets);
#define KV4_STORE(L)                                                                                                       \
    if (lanes == L) QIL_DISPATCH_2(act, weight, qil_launch_chained(kv4_store_kernel<T, W, L>, grid, dim3(32 * STORE_WARPS), 0, stream, a))
    KV4_STORE(4);
    KV4_STORE(8);
    KV4_STORE(16);
    KV4_STORE(32);
    QIL_CHECK_LAUNCH();
}

// ------------------------------------------------------------------ rows back
// A warp: a run of 8 positions of a head's keys or values, groups one after the other: lane (position lane / 4, word lane % 4 of the
// group), 8 elements.  A group of the run is 128 neighbouring bytes.  info: (table row, first position, positions, first page of out)
// a segment; rows of positions without a page are zeros.
static constexpr int READ_WARPS = 8;
// element I of a word of codes as float, exact
template <int I> __device__ __forceinline__ float code_float(unsigned word) {
    return __uint_as_float((word >> (4 * I) & 15u) | 0x4b000000u) - 8388608.f;
}
__device__ __forceinline__ void eight_values(unsigned word, float s, float m, float (&v)[8]) {
    v[0] = fmaf(s, code_float<0>(word), m); v[1] = fmaf(s, code_float<1>(word), m);
    v[2] = fmaf(s, code_float<2>(word), m); v[3] = fmaf(s, code_float<3>(word), m);
    v[4] = fmaf(s, code_float<4>(word), m); v[5] = fmaf(s, code_float<5>(word), m);
    v[6] = fmaf(s, code_float<6>(word), m); v[7] = fmaf(s, code_float<7>(word), m);
}
template <typename T>
__global__ void __launch_bounds__(32 * READ_WARPS)
kv4_read_kernel(const uint8_t* __restrict__ pages, const Kv4Table table, const int* __restrict__ info,
                T* __restrict__ out, int out_pages, int out_page_size, int kv_heads, int dim) {
    qil_wait_for_producer();
    qil_release_consumer();
    const int4 mine = reinterpret_cast<const int4*>(info)[blockIdx.z];
    const int row = mine.x, first = mine.y, count = mine.z, out_first = mine.w;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, groups = dim / KV4_GROUP;
    const int plane = blockIdx.y / kv_heads, head = blockIdx.y % kv_heads;
    // runs are of the pages' positions; a segment may begin inside one
    const int pos = (first / 8 + blockIdx.x * READ_WARPS + warp) * 8 + (lane >> 2), index = pos - first;
    if (index < 0 || index >= count) return;
    const int out_page = out_first + index / out_page_size;
    if (out_page < 0 || out_page >= out_pages) return;
    const int page = table.page(row, pos);
    T* dst = out + ((((size_t)out_page * 2 + plane) * kv_heads + head) * out_page_size + index % out_page_size) * dim + (lane & 3) * 8;
    if (page < 0) {
        const float none[8] = {};
        for (int g = 0; g < groups; ++g) store8(dst + g * KV4_GROUP, none);
        return;
    }
    const int slot = pos % table.page_size;
    const uint8_t* run = pages + kv4_run_at(page, plane, head, slot, kv_heads, table.page_size, groups);
    const uint8_t* codes = run + kv4_code_at(0, slot) + (lane & 3) * 4;
    const uint8_t* pairs = run + kv4_pair_at(0, slot, groups);
#pragma unroll 4
    for (int g = 0; g < groups; ++g) {
        float v[8];
        const unsigned pair = *reinterpret_cast<const unsigned*>(pairs + 4 * g);
        eight_values(*reinterpret_cast<const unsigned*>(codes + g * 128), kv4_step(pair), kv4_base(pair), v);
        store8(dst + g * KV4_GROUP, v);
    }
}

struct Kv4ReadCall {
    const void *pages, *block_table, *info;
    void* out;
    cudaStream_t stream;
    int table_height, table_width, segments, longest, out_pages, out_page_size, kv_heads, dim, page_size, num_pages, act;
};
extern "C" int qil_kv4_read(const void* packed) {
    const auto [pages, block_table, info, out, stream, table_height, table_width, segments, longest, out_pages, out_page_size, kv_heads, dim, page_size,
                num_pages, act] = kv4_call<Kv4ReadCall>(packed);
    if (segments <= 0 || longest <= 0) return 0;
    if (dim <= 0 || dim > KV4_MAX_DIM || dim % KV4_GROUP) QIL_REFUSE("head sizes 32, 64, ..., %d, not %d", KV4_MAX_DIM, dim);
    if (page_size <= 0 || page_size % 8 || out_page_size <= 0) QIL_REFUSE("pages of a multiple of 8 positions, not %d", page_size);
    if (kv_heads <= 0 || 2 * kv_heads > 65535 || segments > 65535) QIL_REFUSE("%d kv heads, %d segments", kv_heads, segments);
    const dim3 grid((longest / 8 + 2 + READ_WARPS - 1) / READ_WARPS, 2 * kv_heads, segments);          // a segment may begin and end inside a run
    QIL_DISPATCH_1(act, qil_launch_chained(kv4_read_kernel<T>, grid, dim3(32 * READ_WARPS), 0, stream, (const uint8_t*)pages,
                                           Kv4Table{(const int*)block_table, table_height, table_width, page_size, num_pages}, (const int*)info,
                                           (T*)out, out_pages, out_page_size, kv_heads, dim));
    QIL_CHECK_LAUNCH();
}

// ------------------------------------------------------------------ a portion's context in 16 bits
static constexpr int SPREAD_PAGE = 64;
struct Kv4Spread {
    const uint8_t* pages;
    Kv4Table table;
    const int* info;                // [segments][4]: table row, the segment's first position, its end, first page of rows
    __half* rows;                   // [page][2][kv head][64][dim]: keys, then values
    float* factors;                 // [page][2][kv head]: what the page's rows are to be multiplied by
    int* value_marks;               // [page][kv head]
    unsigned char* marks;           // [page][kv head][64]
    int kv_heads, dim, window, least;
    int beside;                     // the kernel before this one attends to the same step's short segments
};
// The power of two that brings `largest` into [256, 512) (2^126 at most), and its inverse.  A group's largest value may lie beyond float32,
// its step being rounded up: then 2^-119 brings it next to 512.
__device__ __forceinline__ float bring_up(float largest, float& up) {
    const int e = min(__float_as_int(largest) >> 23, 254);            // 0 of zero and of the smallest numbers
    const int by = min(135 - e, 126);
    up = __int_as_float((127 + by) << 23);
    return __int_as_float((127 - by) << 23);
}
__device__ __forceinline__ unsigned two_halves(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ void store8_half(__half* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(two_halves(v[0], v[1]), two_halves(v[2], v[3]), two_halves(v[4], v[5]), two_halves(v[6], v[7]));
}

// A block: a page of 64 positions of a head's keys or values, a run of 8 a warp (as in kv4_read).
template <int GROUPS>
__global__ void __launch_bounds__(32 * READ_WARPS) kv4_spread_kernel(const Kv4Spread a) {
    __shared__ float largest_of[READ_WARPS];
    // The attention to short segments writes nothing that is read or written here, and all its blocks have seen the end of what came before
    // it when the first of this kernel's starts: so the two run side by side, and the end of this one, which the next kernel waits for, waits
    // for that one's (12 single tokens behind up to 3000 and a portion of 509 behind 6001: 108.7 -> 106.6 us, the faster join of splits in it).
    if (!a.beside) qil_wait_for_producer();
    qil_release_consumer();
    constexpr int dim = GROUPS * KV4_GROUP;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int4 mine = reinterpret_cast<const int4*>(a.info)[blockIdx.z];
    const int plane = blockIdx.y / a.kv_heads, head = blockIdx.y % a.kv_heads;
    const int page0 = blockIdx.x * SPREAD_PAGE;
    if (mine.z - mine.y < a.least || page0 >= mine.z || (a.window > 0 && page0 + SPREAD_PAGE <= mine.y + 1 - a.window)) {       // nobody will look
        qil_wait_for_producer();
        return;
    }
    const int slot_out = warp * 8 + (lane >> 2), pos = page0 + slot_out;
    const size_t at = (size_t)(mine.w + blockIdx.x) * a.kv_heads + head;
    __half* dst = a.rows + ((((size_t)(mine.w + blockIdx.x) * 2 + plane) * a.kv_heads + head) * SPREAD_PAGE + slot_out) * dim + (lane & 3) * 8;
    const int page = pos < mine.z ? a.table.page(mine.x, pos) : -1;
    unsigned codes[GROUPS], pairs[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) codes[g] = pairs[g] = 0u;
    if (page >= 0) {
        const int slot = pos % a.table.page_size;
        const uint8_t* run = a.pages + kv4_run_at(page, plane, head, slot, a.kv_heads, a.table.page_size, GROUPS);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            codes[g] = *reinterpret_cast<const unsigned*>(run + kv4_code_at(g, slot) + (lane & 3) * 4);
            pairs[g] = *reinterpret_cast<const unsigned*>(run + kv4_pair_at(g, slot, GROUPS));
        }
    }
    unsigned nan = 0u;
    float largest = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        const float s = kv4_step(pairs[g]), m = kv4_base(pairs[g]);
        if (plane == 1 && !(s == s)) {
            nan |= 1u << g;
            pairs[g] = 0u;
        } else {
            largest = fmaxf(largest, fmaxf(fabsf(m), fabsf(fmaf(15.f, s, m))));            // NaN is left out
        }
    }
    largest = warp_max(largest);
    if (lane == 0) largest_of[warp] = largest;
    const int any = __syncthreads_or(nan != 0u);
    largest = largest_of[0];
#pragma unroll
    for (int w = 1; w < READ_WARPS; ++w) largest = fmaxf(largest, largest_of[w]);
    float up;
    const float factor = bring_up(largest, up);
    if (threadIdx.x == 0) a.factors[((size_t)(mine.w + blockIdx.x) * 2 + plane) * a.kv_heads + head] = factor;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        float v[8];
        eight_values(codes[g], kv4_step(pairs[g]) * up, kv4_base(pairs[g]) * up, v);          // exact, and nothing of it is infinite
        store8_half(dst + g * KV4_GROUP, v);
    }
    if (plane == 1) {
        if (threadIdx.x == 0) a.value_marks[at] = any;
        if (any && (lane & 3) == 0) a.marks[at * SPREAD_PAGE + slot_out] = (unsigned char)nan;
    }
    qil_wait_for_producer();
}

struct Kv4SpreadCall {
    const void *pages, *block_table, *info;
    void *rows, *factors, *value_marks, *marks;
    cudaStream_t stream;
    int table_height, table_width, segments, width, kv_heads, dim, page_size, num_pages, window, least, beside;
};
extern "C" int qil_kv4_spread(const void* packed) {
    const auto [pages, block_table, info, rows, factors, value_marks, marks, stream, table_height, table_width, segments, width, kv_heads, dim,
                page_size, num_pages, window, least, beside] = kv4_call<Kv4SpreadCall>(packed);
    if (segments <= 0 || width <= 0) return 0;
    if (dim <= 0 || dim > 128 || dim % KV4_GROUP) QIL_REFUSE("head sizes 32, 64, 96, 128, not %d", dim);
    if (page_size <= 0 || page_size % 8) QIL_REFUSE("pages of a multiple of 8 positions, not %d", page_size);
    if (kv_heads <= 0 || 2 * kv_heads > 65535 || segments >= 65535) QIL_REFUSE("%d kv heads, %d segments", kv_heads, segments);
    const Kv4Spread a = {(const uint8_t*)pages, {(const int*)block_table, table_height, table_width, page_size, num_pages}, (const int*)info,
                         (__half*)rows, (float*)factors, (int*)value_marks, (unsigned char*)marks, kv_heads, dim, window, least, beside};
    const dim3 grid(width, 2 * kv_heads, segments);
    void (*kernel)(Kv4Spread) = dim == 32 ? kv4_spread_kernel<1> : dim == 64 ? kv4_spread_kernel<2> : dim == 96 ? kv4_spread_kernel<3> : kv4_spread_kernel<4>;
    qil_launch_chained(kernel, grid, dim3(32 * READ_WARPS), 0, stream, a);
    QIL_CHECK_LAUNCH();
}

extern "C" int qil_kv4_call_bytes(int which) { return which == 0 ? sizeof(Kv4StoreCall) : which == 1 ? sizeof(Kv4ReadCall) : sizeof(Kv4SpreadCall); }
