// Attention over the quantized key / value cache (kv_format.hpp has the format).
//
// Row i of the n rows of a sequence of L cached tokens stands at p = L - n + i.  With s_j =
// cap(scale q.k_j) + slope (j - p) over the tokens j <= p (causal) and j > p - window,
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),
// computed in one walk over the tokens with a running maximum m and sum; a row that no token is
// visible to is zero.  All query heads of a cached head are rows of one matrix, so a key or value is
// read and decoded once for them.
//
// Both products run on v_mfma_f32_16x16x32_bf16, transposed: S^T = K Q^T leaves a lane the scores of
// one row (column lane % 16) and of 4 tokens of a chunk of 16 (rows 4 (lane / 16) ..), and two
// chunks give it the 8 tokens that the second product, O^T = V^T P^T, wants of it as an operand: the
// probabilities never leave its registers.  Keys and values are exact in bfloat16.  Queries are
// taken apart into a sum of TERMS bfloat16 numbers, exactly (1 from bfloat16, 2 from float16, 3
// from float32), and probabilities likewise, where one term is a rounding to bfloat16's 8 bits (half
// a step, 2^-8 of a weight, as the rounding of a bfloat16 output is; the weights' errors mostly
// cancel), two hold 16 bits and three 24.
#include "kv_format.hpp"
#include "internal.hpp"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxSplits = 64;

struct AttnArgs {
    const uint8_t* data;
    icx::KvLayout l;
    int pages, page_size;
    const void* q;
    int64_t q_row, q_head;  // strides, elements
    void* out;
    int64_t o_row, o_head;
    const int32_t* table;
    int64_t table_stride;
    int width;
    const int32_t* lengths;
    const int32_t* starts;  // null: one row a sequence
    int batch, group, heads_q, max_rows, rows_total;
    float scale, softcap;
    int window, causal;
    const float* slopes;
    int row_tiles, splits;
    float* part;   // [splits][rows_total * heads_q][D] sums of exp(s - m) v
    float2* ml;    // [splits][rows_total * heads_q] (m, in powers of two; sum of exp)
};

// The rows and tokens of one sequence, from the device's own lengths: what is out of range is cut to it.
struct Sequence {
    int start, rows, len;  // rows: those that are done, at most max_rows
    int base;              // position of the first row
};
__device__ __forceinline__ Sequence sequence(const AttnArgs& a, int b) {
    Sequence s;
    s.start = a.starts ? a.starts[b] : b;
    int n = 0;
    if (s.start >= 0 && s.start <= a.rows_total) n = a.starts ? max(0, min(a.starts[b + 1], a.rows_total) - s.start) : 1;
    s.rows = min(n, a.max_rows);
    s.len = max(0, min(a.lengths[b], a.width * a.page_size));
    s.base = s.len - n;
    return s;
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// v[0..7] as a sum of TERMS packed bfloat16 operands.
template <int TERMS>
__device__ __forceinline__ void split_terms(const float (&v)[8], bf16x8 (&t)[TERMS]) {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
    for (int n = 0; n < TERMS; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const __bf16 h = (__bf16)r[e];
            t[n][e] = h;
            if (n + 1 < TERMS) r[e] -= (float)h;
        }
}

// tanh to a few ulps: away from 0 through exp, near it by its series (exp's form loses digits there).
__device__ __forceinline__ float tanh_f32(float x) {
    const float y = fabsf(x);
    const float z = y * y;
    const float near = y * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    const float e = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e));
    const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f);
    return copysignf(y < 0.25f ? near : far, x);
}

// The codes and scales of 32 tokens (two chunks) of one cached head, as a lane's operands need them.
// GM: blocks of 32 that there is room for; EXACT: G == GM.
template <int BITS, int GM>
struct Tile {
    uint32_t k[2][GM * BITS / 4];
    uint32_t v[2][GM * BITS / 4];
    uint32_t ks[2][GM <= 4 ? 1 : 2];  // the lane's keys' scales, a byte for each of its blocks
    uint32_t vs[2][GM];               // the values' scales of its 4 tokens, by block
};

template <int N>
__device__ __forceinline__ void load_dwords(const uint8_t* p, uint32_t (&d)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u32x4 w = reinterpret_cast<const u32x4*>(p)[i];
            d[4 * i] = w[0];
            d[4 * i + 1] = w[1];
            d[4 * i + 2] = w[2];
            d[4 * i + 3] = w[3];
        }
    } else {
        static_assert(N == 2, "");
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        d[0] = w.x;
        d[1] = w.y;
    }
}

template <int BITS, int GM, bool EXACT>
__device__ __forceinline__ void load_chunk(const uint8_t* c, int G, int lane, Tile<BITS, GM>& t, int n) {
    const int lr = lane & 15, j = lane >> 4;
    const uint8_t* kp = c + (lr * 4 + j) * G * BITS;
    const uint8_t* vp = c + icx::kv_codes(G, BITS) + (j * 16 + lr) * G * BITS;
    const uint8_t* sp = c + icx::kv_key_scales(G, BITS) + lr * G;
    const uint8_t* vq = c + icx::kv_value_scales(G, BITS) + j * 4 * G;
    if constexpr (EXACT) {
        load_dwords(kp, t.k[n]);
        load_dwords(vp, t.v[n]);
        load_dwords(vq, t.vs[n]);
        if constexpr (GM == 2) t.ks[n][0] = sp[j >> 1];
        else if constexpr (GM == 4) t.ks[n][0] = sp[j];
        else t.ks[n][0] = *reinterpret_cast<const uint16_t*>(sp + 2 * j);
    } else {
        static_assert(GM == 8, "");
        t.ks[n][0] = t.ks[n][1] = 0;
#pragma unroll
        for (int i = 0; i < GM; ++i) {
            if (i >= G) break;
            if (BITS == 4) {
                t.k[n][i] = reinterpret_cast<const uint32_t*>(kp)[i];
                t.v[n][i] = reinterpret_cast<const uint32_t*>(vp)[i];
            } else {
                const uint2 x = reinterpret_cast<const uint2*>(kp)[i], y = reinterpret_cast<const uint2*>(vp)[i];
                t.k[n][2 * i % (GM * BITS / 4)] = x.x;
                t.k[n][(2 * i + 1) % (GM * BITS / 4)] = x.y;
                t.v[n][2 * i % (GM * BITS / 4)] = y.x;
                t.v[n][(2 * i + 1) % (GM * BITS / 4)] = y.y;
            }
            t.vs[n][i] = reinterpret_cast<const uint32_t*>(vq)[i];
            t.ks[n][i >> 2] |= (uint32_t)sp[(j * G + i) >> 2] << (8 * (i & 3));  // the block of step i
        }
    }
}

// Keys' operand of step i (values j D / 4 + 8 i .. + 7 of the lane's token).
template <int BITS, int GM, bool EXACT>
__device__ __forceinline__ bf16x8 key_operand(const Tile<BITS, GM>& t, int n, int i) {
    float s;
    if constexpr (!EXACT) s = icx::scale_of(t.ks[n][i >> 2], i & 3);
    else if constexpr (GM == 8) s = icx::scale_of(t.ks[n][0], i >> 2);
    else s = icx::scale_of(t.ks[n][0], 0);
    u32x4 w;
    if constexpr (BITS == 4) {
        w[0] = icx::decode2<4, 0>(t.k[n][i], s);
        w[1] = icx::decode2<4, 1>(t.k[n][i], s);
        w[2] = icx::decode2<4, 2>(t.k[n][i], s);
        w[3] = icx::decode2<4, 3>(t.k[n][i], s);
    } else {
        const uint32_t x = t.k[n][2 * i], y = t.k[n][2 * i + 1];
        w[0] = icx::decode2<8, 0>(x, s);
        w[1] = icx::decode2<8, 1>(x, s);
        w[2] = icx::decode2<8, 0>(y, s);
        w[3] = icx::decode2<8, 1>(y, s);
    }
    return __builtin_bit_cast(bf16x8, w);
}

// Values' operands of block g: rows d = 32 g + lane % 16 (lo) and 16 further (hi), the lane's 8 tokens.
template <int BITS, int GM>
__device__ __forceinline__ void value_operands(const Tile<BITS, GM>& t, int g, bf16x8& lo, bf16x8& hi) {
    u32x4 l, h;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        uint32_t p[4];
        const uint32_t s = t.vs[n][g];
        if constexpr (BITS == 4) {
            const uint32_t w = t.v[n][g];
            p[0] = icx::decode2<4, 0>(w, icx::scale_of(s, 0));
            p[1] = icx::decode2<4, 1>(w, icx::scale_of(s, 1));
            p[2] = icx::decode2<4, 2>(w, icx::scale_of(s, 2));
            p[3] = icx::decode2<4, 3>(w, icx::scale_of(s, 3));
        } else {
            const uint32_t w = t.v[n][2 * g], x = t.v[n][2 * g + 1];
            p[0] = icx::decode2<8, 0>(w, icx::scale_of(s, 0));
            p[1] = icx::decode2<8, 1>(w, icx::scale_of(s, 1));
            p[2] = icx::decode2<8, 0>(x, icx::scale_of(s, 2));
            p[3] = icx::decode2<8, 1>(x, icx::scale_of(s, 3));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[2 * n + e] = __builtin_amdgcn_perm(p[2 * e + 1], p[2 * e], 0x05040100u);
            h[2 * n + e] = __builtin_amdgcn_perm(p[2 * e + 1], p[2 * e], 0x07060302u);
        }
    }
    lo = __builtin_bit_cast(bf16x8, l);
    hi = __builtin_bit_cast(bf16x8, h);
}

// What a tile of 32 tokens from t0 needs beside its data.
struct Place {
    const uint8_t* c[2];
    bool there[2];
};
__device__ __forceinline__ Place place(const AttnArgs& a, const int32_t* row, const uint8_t* head, int t0) {
    Place p;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int chunk = (t0 >> 4) + n;
        const int at = min(chunk / a.l.chunks, a.width - 1);
        const int page = row[at];
        p.there[n] = page >= 0 && page < a.pages;
        p.c[n] = head + (int64_t)(p.there[n] ? page : 0) * a.l.page_bytes + (int64_t)(chunk % a.l.chunks) * a.l.chunk_bytes;
    }
    return p;
}

// One block: 16 rows (row tile rt) of one cached head of one sequence, one share of its tokens; the
// four waves take tiles of 32 tokens in turn and are joined at the end.
constexpr int kWaves = 4;

template <int BITS, int TERMS, int GM, bool EXACT, typename T>
__global__ void __launch_bounds__(64 * kWaves) kv_attention_rows_kernel(AttnArgs a) {
    extern __shared__ float smem[];  // [waves][16 rows][D + 4] then (m, l) [waves][16]
    const int G = EXACT ? GM : a.l.G, D = 32 * G;
    const int lane = threadIdx.x & 63, lr = lane & 15, j = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int x = blockIdx.x;
    const int split = x % a.splits;
    x /= a.splits;
    const int rt = x % a.row_tiles;
    x /= a.row_tiles;
    const int h = x % a.l.heads, b = x / a.l.heads;
    const Sequence sq = sequence(a, b);
    const int rows = sq.rows * a.group;
    if (rt * 16 >= rows) return;
    const int first = rt * 16 / a.group, last = min(rt * 16 + 15, rows - 1) / a.group;
    const int base = sq.base;
    const int end = a.causal ? max(0, min(sq.len, base + last + 1)) : sq.len;
    const int begin = a.window > 0 ? max(0, base + first - a.window + 1) : 0;
    // every row sees every token of [full_begin, full_end)
    const int full_end = a.causal ? min(sq.len, base + first + 1) : sq.len;
    const int full_begin = a.window > 0 ? base + last - a.window + 1 : 0;
    const int tile0 = begin >> 5, tiles = max(0, ((end + 31) >> 5) - tile0);
    const int share = max(kWaves, (tiles + a.splits - 1) / a.splits);
    const int from = min(tiles, split * share), to = min(tiles, from + share);

    // the lane's row
    const int r = rt * 16 + lr;
    const bool row_there = r < rows;
    const int tok = min(r, rows - 1) / a.group, hq = h * a.group + min(r, rows - 1) % a.group;
    const int p = base + tok;
    const int lowest = a.window > 0 ? p - a.window : -1;  // a token is seen above it
    const int highest = a.causal ? min(p, sq.len - 1) : sq.len - 1;
    const float slope = a.slopes ? a.slopes[hq] * kLog2e : 0.0f;
    const float c = a.scale * kLog2e, cap = a.softcap * kLog2e, incap = a.softcap > 0.0f ? a.scale / a.softcap : 0.0f;

    bf16x8 qf[GM][TERMS];
    {
        const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)(sq.start + tok) * a.q_row + (int64_t)hq * a.q_head + j * 8 * G;
#pragma unroll
        for (int i = 0; i < GM; ++i) {
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if ((EXACT || i < G) && row_there) icx::load_f32(qp + 8 * i, v);
            split_terms<TERMS>(v, qf[i]);
        }
    }

    f32x4 acc[2 * GM];
#pragma unroll
    for (int i = 0; i < 2 * GM; ++i) acc[i] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;

    const uint8_t* head = a.data + (int64_t)h * a.l.head_bytes;
    const int32_t* table = a.table + b * a.table_stride;
    Tile<BITS, GM> t;
    for (int i = from + wid; i < to; i += kWaves) {
        const int t0 = (tile0 + i) * 32;
        const Place pl = place(a, table, head, t0);
        load_chunk<BITS, GM, EXACT>(pl.c[0], G, lane, t, 0);
        load_chunk<BITS, GM, EXACT>(pl.c[1], G, lane, t, 1);
        const bool edge = t0 < full_begin || t0 + 32 > full_end || !pl.there[0] || !pl.there[1];

        f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int e = 0; e < GM; ++e) {
            if (!EXACT && e >= G) break;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const bf16x8 k = key_operand<BITS, GM, EXACT>(t, n, e);
#pragma unroll
                for (int u = 0; u < TERMS; ++u) s[n] = mfma(k, qf[e][u], s[n]);
            }
        }
        // scores in powers of two
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = a.softcap > 0.0f ? cap * tanh_f32(s[e >> 2][e & 3] * incap) : s[e >> 2][e & 3] * c;
        if (a.slopes) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = fmaf(slope, (float)(t0 + 16 * (e >> 2) + 4 * j + (e & 3) - p), w[e]);
        }
        uint32_t spoilt = 0;  // blocks whose NaN the row sees (edge tiles)
        if (edge) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int at = t0 + 16 * (e >> 2) + 4 * j + (e & 3);
                const bool seen = at > lowest && at <= highest && pl.there[e >> 2];
                if (!seen) w[e] = -INFINITY;
                // A weight of zero does not take a NaN out of the product: a NaN block counts as zeros
                // there, and reaches the rows that see it by hand.
#pragma unroll
                for (int g = 0; g < GM; ++g) {
                    if (!EXACT && g >= G) break;
                    const uint32_t byte = 255u << (8 * (e & 3));
                    if ((t.vs[e >> 2][g] & byte) == byte) {
                        t.vs[e >> 2][g] &= ~byte;
                        if (seen) spoilt |= 1u << g;
                    }
                }
            }
            spoilt |= (uint32_t)__shfl_xor((int)spoilt, 16, 64);
            spoilt |= (uint32_t)__shfl_xor((int)spoilt, 32, 64);
        }
        float top = w[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, w[e]);
        // The running maximum moves only when a score passes it by 2^8: until then the weights stay
        // below 256 and the sums need no rescaling.
        if (__any(top > m + 8.0f)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float next = fmaxf(m, top);
            const float f = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= f;
#pragma unroll
            for (int e = 0; e < 2 * GM; ++e) acc[e] *= f;
        }
        const float mu = m == -INFINITY ? 0.0f : m;
        float pr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            pr[e] = __builtin_amdgcn_exp2f(w[e] - mu);
            l += pr[e];
        }
        bf16x8 pf[TERMS];
        split_terms<TERMS>(pr, pf);
#pragma unroll
        for (int g = 0; g < GM; ++g) {
            if (!EXACT && g >= G) break;
            bf16x8 lo, hi;
            value_operands<BITS, GM>(t, g, lo, hi);
#pragma unroll
            for (int u = 0; u < TERMS; ++u) {
                acc[2 * g] = mfma(lo, pf[u], acc[2 * g]);
                acc[2 * g + 1] = mfma(hi, pf[u], acc[2 * g + 1]);
            }
        }
        if (spoilt) {
#pragma unroll
            for (int g = 0; g < GM; ++g)
                if (spoilt >> g & 1) {
                    acc[2 * g] += __builtin_nanf("");
                    acc[2 * g + 1] += __builtin_nanf("");
                }
        }
    }

    // join the waves
    const int held = min(16, rows - rt * 16), stride = D + 4;
    float2* ml = reinterpret_cast<float2*>(smem + kWaves * held * stride);
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (lane < held) ml[wid * 16 + lane] = make_float2(m, l);
    if (lr < held) {
        float* o = smem + (wid * held + lr) * stride + 4 * j;
#pragma unroll
        for (int e = 0; e < 2 * GM; ++e)
            if (EXACT || e < 2 * G) *reinterpret_cast<f32x4*>(o + 16 * e) = acc[e];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < held * (D / 4); e += 64 * kWaves) {
        const int row = e / (D / 4), d = e % (D / 4) * 4;
        float top = ml[row].x;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, ml[w * 16 + row].x);
        const float mu = top == -INFINITY ? 0.0f : top;
        f32x4 sum = {0, 0, 0, 0};
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(ml[w * 16 + row].x - mu);
            total += f * ml[w * 16 + row].y;
            sum += f * *reinterpret_cast<const f32x4*>(smem + (w * held + row) * stride + d);
        }
        const int rr = rt * 16 + row, tk = rr / a.group, qh = h * a.group + rr % a.group;
        const int64_t at = (int64_t)(sq.start + tk) * a.heads_q + qh;
        if (a.splits > 1) {
            *reinterpret_cast<f32x4*>(a.part + ((int64_t)split * a.rows_total * a.heads_q + at) * D + d) = sum;
            if (d == 0) a.ml[(int64_t)split * a.rows_total * a.heads_q + at] = make_float2(top, total);
        } else {
            const bool any = !(total == 0.0f && top == -INFINITY);  // no token: zero
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = any ? sum[k] / total : 0.0f;
            icx::store_f32(reinterpret_cast<T*>(a.out) + (int64_t)(sq.start + tk) * a.o_row + (int64_t)qh * a.o_head + d, v);
        }
    }
}

// Joins the shares of every row: a wave a row.
template <typename T>
__global__ void __launch_bounds__(256) kv_attention_join_kernel(AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int D = 32 * a.l.G;
    const int hq = (int)(id % a.heads_q);
    const int64_t x = id / a.heads_q;
    const int tok = (int)(x % a.max_rows);
    const int64_t b = x / a.max_rows;
    if (b >= a.batch) return;
    const Sequence sq = sequence(a, (int)b);
    if (tok >= sq.rows) return;
    const int64_t at = (int64_t)(sq.start + tok) * a.heads_q + hq, all = (int64_t)a.rows_total * a.heads_q;
    float top = -INFINITY;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.ml[s * all + at].x);
    const float mu = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    for (int s = 0; s < a.splits; ++s) {
        const float2 e = a.ml[s * all + at];
        total += __builtin_amdgcn_exp2f(e.x - mu) * e.y;
    }
    const bool any = !(total == 0.0f && top == -INFINITY);
    for (int d = 4 * lane; d < D; d += 256) {
        f32x4 sum = {0, 0, 0, 0};
        for (int s = 0; s < a.splits; ++s) {
            const float f = __builtin_amdgcn_exp2f(a.ml[s * all + at].x - mu);
            sum += f * *reinterpret_cast<const f32x4*>(a.part + (s * all + at) * D + d);
        }
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = any ? sum[k] / total : 0.0f;
        icx::store_f32(reinterpret_cast<T*>(a.out) + (int64_t)(sq.start + tok) * a.o_row + (int64_t)hq * a.o_head + d, v);
    }
}

template <int BITS, int TERMS, typename T>
void launch_rows(unsigned blocks, hipStream_t s, const AttnArgs& a) {
    const int D = 32 * a.l.G;
    const size_t held = (size_t)std::min(16, a.max_rows * a.group);
    const size_t lds = kWaves * held * (D + 4) * 4 + kWaves * 16 * 8;
    switch (a.l.G) {
        case 2: kv_attention_rows_kernel<BITS, TERMS, 2, true, T><<<blocks, 64 * kWaves, lds, s>>>(a); break;
        case 4: kv_attention_rows_kernel<BITS, TERMS, 4, true, T><<<blocks, 64 * kWaves, lds, s>>>(a); break;
        case 8: kv_attention_rows_kernel<BITS, TERMS, 8, true, T><<<blocks, 64 * kWaves, lds, s>>>(a); break;
        default: kv_attention_rows_kernel<BITS, TERMS, 8, false, T><<<blocks, 64 * kWaves, lds, s>>>(a); break;
    }
}

// How the call is cut: row tiles of 16 and shares of the tokens.
struct Plan {
    int row_tiles, splits;
    size_t blocks, part_bytes, ml_bytes;
};
Plan plan_of(const icx_kv_cache& c, const icx_kv_attention& a) {
    Plan p;
    const size_t group = (size_t)(a.q_heads / c.kv_heads);
    p.row_tiles = (int)icx::cdiv((size_t)a.max_rows * group, 16);
    const size_t one = (size_t)a.batch * c.kv_heads * p.row_tiles;
    const size_t tokens = (size_t)a.table_width * c.page_size;
    const size_t want = icx::cdiv((size_t)icx::num_cus() * 8, std::max<size_t>(one, 1));
    p.splits = (int)std::max<size_t>(1, std::min({want, icx::cdiv(tokens, 256), (size_t)kMaxSplits}));
    p.blocks = one * p.splits;
    const size_t rows = (size_t)a.rows * a.q_heads;
    p.part_bytes = p.splits > 1 ? icx::align_up((size_t)p.splits * rows * c.head_size * 4, 256) : 0;
    p.ml_bytes = p.splits > 1 ? (size_t)p.splits * rows * 8 : 0;
    return p;
}

int check_attention(const icx_kv_cache* c, const icx_kv_attention* a, const char* who) {
    int rc = icx::check_kv_cache(c, who);
    if (rc) return rc;
    if (!a) ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: null arguments", who);
    if (!icx::is_float_kind(a->dtype))
        ICX_FAIL(ICX_ERR_DTYPE, "%s: dtype %d unsupported (must be Float32, Float16 or BFloat16)", who, a->dtype);
    if (a->q_heads < 1 || a->q_heads % c->kv_heads)
        ICX_FAIL(ICX_ERR_SHAPE, "%s: %d query heads over %d cached ones", who, a->q_heads, c->kv_heads);
    if (a->batch < 0 || a->rows < 0 || a->table_width < 0 || a->max_rows < 0)
        ICX_FAIL(ICX_ERR_SHAPE, "%s: negative size", who);
    // (positions, and a window's distance from them, stay within 32 bits)
    if ((int64_t)a->table_width * c->page_size > 0x40000000 || a->rows > 0x40000000)
        ICX_FAIL(ICX_ERR_SHAPE, "%s: %lld tokens a sequence, %d rows are too many", who,
                 (long long)a->table_width * c->page_size, a->rows);
    if (!a->q_starts && a->rows != a->batch)
        ICX_FAIL(ICX_ERR_SHAPE, "%s: without q_starts there is one row a sequence (%d rows, %d sequences)", who, a->rows, a->batch);
    if (!(a->softcap >= 0.0f) || a->window < 0)
        ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: softcap %g and window %d must not be negative", who, (double)a->softcap, a->window);
    return ICX_OK;
}

}  // namespace

extern "C" size_t icx_kv_cache_attention_workspace_size(const icx_kv_cache* cache, const icx_kv_attention* args) {
    icx::clear_error();
    if (check_attention(cache, args, "KvCacheAttention")) return 0;
    const Plan p = plan_of(*cache, *args);
    return p.part_bytes + p.ml_bytes;
}

extern "C" int icx_kv_cache_attention(icx_stream_t stream, const icx_kv_cache* cache, const icx_kv_attention* args, void* ws,
                                      size_t ws_bytes) {
    icx::clear_error();
    const char* who = "KvCacheAttention";
    int rc = check_attention(cache, args, who);
    if (rc) return rc;
    if (args->rows == 0 || args->batch == 0 || args->max_rows == 0) return ICX_OK;
    if (!args->q || !args->out || !args->lengths || (!args->page_table && args->table_width))
        ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: null q, out, page_table or lengths", who);
    const Plan p = plan_of(*cache, *args);
    if (p.blocks * 64 * kWaves > 0xffffffffull || (uint64_t)args->batch * args->max_rows * args->q_heads * 64 > 0xffffffffull)
        ICX_FAIL(ICX_ERR_UNSUPPORTED, "%s: %d sequences of up to %d rows are too many for a launch", who, args->batch, args->max_rows);
    if (p.part_bytes && (!ws || ws_bytes < p.part_bytes + p.ml_bytes))
        ICX_FAIL(ICX_ERR_WORKSPACE, "%s: workspace of %zu bytes needed (got %zu)", who, p.part_bytes + p.ml_bytes, ws_bytes);
    AttnArgs a{};
    a.data = reinterpret_cast<const uint8_t*>(cache->data);
    a.l = icx::kv_layout(*cache);
    a.pages = (int)cache->pages;
    a.page_size = cache->page_size;
    a.q = args->q;
    a.q_row = args->q_row_stride;
    a.q_head = args->q_head_stride;
    a.out = args->out;
    a.o_row = args->out_row_stride;
    a.o_head = args->out_head_stride;
    a.table = args->page_table;
    a.table_stride = args->table_stride;
    a.width = args->table_width;
    a.lengths = args->lengths;
    a.starts = args->q_starts;
    a.batch = args->batch;
    a.group = args->q_heads / cache->kv_heads;
    a.heads_q = args->q_heads;
    a.max_rows = args->max_rows;
    a.rows_total = args->rows;
    a.scale = args->scale;
    a.softcap = args->softcap;
    a.window = args->window < args->table_width * cache->page_size ? args->window : 0;  // 0: every token
    a.causal = args->causal;
    a.slopes = args->slopes;
    a.row_tiles = p.row_tiles;
    a.splits = p.splits;
    a.part = reinterpret_cast<float*>(ws);
    a.ml = reinterpret_cast<float2*>(reinterpret_cast<char*>(ws) + p.part_bytes);
    const hipStream_t s = (hipStream_t)stream;
    const unsigned blocks = (unsigned)p.blocks;
    const bool four = cache->bits == 4;
    if (args->dtype == ICX_BF16) four ? launch_rows<4, 1, __bf16>(blocks, s, a) : launch_rows<8, 1, __bf16>(blocks, s, a);
    else if (args->dtype == ICX_F16) four ? launch_rows<4, 2, _Float16>(blocks, s, a) : launch_rows<8, 2, _Float16>(blocks, s, a);
    else four ? launch_rows<4, 3, float>(blocks, s, a) : launch_rows<8, 3, float>(blocks, s, a);
    ICX_LAUNCH_CHECK("kv_attention_rows_kernel");
    if (p.splits > 1) {
        const unsigned jb = (unsigned)icx::cdiv((size_t)args->batch * args->max_rows * args->q_heads, 4);
        icx::with_float_type(args->dtype, [&](auto* t) -> int {
            kv_attention_join_kernel<std::remove_pointer_t<decltype(t)>><<<jb, 256, 0, s>>>(a);
            return 0;
        });
        ICX_LAUNCH_CHECK("kv_attention_join_kernel");
    }
    return ICX_OK;
}
