// Writing keys and values into the quantized cache and reading them back (kv_format.hpp has the
// format).
//
// Four lanes share a block of 32 values.  A lane takes 8 consecutive keys (its codes are then a
// whole dword or two of the token's row), and of the values 4 consecutive ones of each half of the
// block, the pairs that a byte of the transposed layout holds.  The conversions are one instruction a
// pair; what bounds the kernels is memory, and how it is reached.  A token alone leaves its values' codes
// in bytes apart, each an access of its own; so for many tokens a wave takes 16 of them and one head, and
// where their slots are a chunk of 16 from its start on, as a prompt's are, the chunk goes through LDS and to
// memory in whole lines (kv_write_chunks_kernel, kv_read_chunks_kernel).
#include <type_traits>

#include "kv_format.hpp"

namespace {

constexpr int kThreads = 256;

struct CacheArgs {
    uint8_t* data;
    icx::KvLayout l;
    int64_t slots_end;  // pages * page_size
    int page_size;
    const void* slots;
    int slots64;
    int64_t tokens;
    const void* k;
    const void* v;
    int64_t k_token, k_head, v_token, v_head;  // strides, elements
    void* k_out;
    void* v_out;
    int64_t units;  // tokens * heads * G
};

__device__ __forceinline__ int64_t slot_of(const CacheArgs& a, int64_t t) {
    return a.slots64 ? reinterpret_cast<const int64_t*>(a.slots)[t] : (int64_t)reinterpret_cast<const int32_t*>(a.slots)[t];
}

__device__ __forceinline__ uint8_t* chunk_of(const CacheArgs& a, int64_t slot, int head, int& t16) {
    const int64_t page = slot / a.page_size;
    const int in = (int)(slot - page * a.page_size);
    t16 = in & 15;
    return a.data + page * a.l.page_bytes + (int64_t)head * a.l.head_bytes + (int64_t)(in >> 4) * a.l.chunk_bytes;
}

// The largest magnitude's bits over the four lanes of a block (NaN above infinity above the rest).
__device__ __forceinline__ uint32_t block_top(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
    return max(m, (uint32_t)__shfl_xor((int)m, 2, 64));
}

// Codes of v[0..7], two a byte (4 bits) or a half (8 bits), pairs in order: the instruction rounds to
// nearest even and, in 4 bits, takes the largest code for what is past it.  In 8 bits that would be
// a NaN, and is kept out by the clamp; only a block whose scale is at its upper end needs it.
template <int BITS>
__device__ __forceinline__ uint2 encode8(float (&v)[8], uint32_t eb) {
    if (eb == 255u) return make_uint2(0u, 0u);
    const float s = __uint_as_float(eb << 23);
    if constexpr (BITS == 4) {
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
        return make_uint2(w, 0u);
    } else {
        typedef short s16x2 __attribute__((ext_vector_type(2)));
        if (eb == 246u) {
            const float top = 448.0f * s;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fminf(fmaxf(v[i], -top), top);
        }
        s16x2 a = {0, 0}, b = {0, 0};
        a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[0], v[1], s, false);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[2], v[3], s, true);
        b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[4], v[5], s, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[6], v[7], s, true);
        return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
    }
}

// A lane's codes, and the block's scales from its first lane, into a chunk.
template <int BITS>
__device__ __forceinline__ void put_codes(uint8_t* c, int G, int t16, int g, int i, uint2 kc, uint2 vc, uint32_t ke, uint32_t ve) {
    uint8_t* kd = c + (t16 * G + g) * 4 * BITS + i * BITS;
    if (BITS == 4) *reinterpret_cast<uint32_t*>(kd) = kc.x;
    else *reinterpret_cast<uint2*>(kd) = kc;
    uint8_t* vd = c + icx::kv_codes(G, BITS) + (((t16 >> 2) * 16 + 4 * i) * G + g) * BITS + (t16 & 3) * (BITS / 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (BITS == 4) vd[e * G * BITS] = (uint8_t)(vc.x >> (8 * e));
        else *reinterpret_cast<uint16_t*>(vd + e * G * BITS) = (uint16_t)((e < 2 ? vc.x : vc.y) >> (16 * (e & 1)));
    }
    if (i == 0) {
        c[icx::kv_key_scales(G, BITS) + t16 * G + g] = (uint8_t)ke;
        c[icx::kv_value_scales(G, BITS) + ((t16 >> 2) * G + g) * 4 + (t16 & 3)] = (uint8_t)ve;
    }
}

template <int BITS, typename T>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(CacheArgs a) {
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t unit = id >> 2;
    const int i = (int)(id & 3);
    const int G = a.l.G;
    // every lane of a block of 32 takes the same way through here
    if (unit >= a.units) return;
    const int g = (int)(unit % G);
    const int64_t th = unit / G;
    const int h = (int)(th % a.l.heads);
    const int64_t t = th / a.l.heads;
    const int64_t slot = slot_of(a, t);
    if (slot < 0 || slot >= a.slots_end) return;
    float k[8], v[8];
    const T* kp = reinterpret_cast<const T*>(a.k) + t * a.k_token + h * a.k_head + 32 * g + 8 * i;
    const T* vp = reinterpret_cast<const T*>(a.v) + t * a.v_token + h * a.v_head + 32 * g + 4 * i;
    icx::load_f32(kp, k);
    {
        float lo[4], hi[4];
        icx::load_f32(vp, lo);
        icx::load_f32(vp + 16, hi);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = lo[e];
            v[2 * e + 1] = hi[e];
        }
    }
    const uint32_t ke = icx::block_exponent<BITS>(block_top(k)), ve = icx::block_exponent<BITS>(block_top(v));
    const uint2 kc = encode8<BITS>(k, ke), vc = encode8<BITS>(v, ve);
    int t16;
    uint8_t* c = chunk_of(a, slot, h, t16);
    put_codes<BITS>(c, G, t16, g, i, kc, vc, ke, ve);
}

__device__ __forceinline__ void unpack(uint32_t w, float& lo, float& hi) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
}

// A lane's values from a chunk, and into the outputs.
template <int BITS>
__device__ __forceinline__ void take_codes(const uint8_t* c, int G, int t16, int g, int i, float (&k)[8], float (&v)[8]) {
    const int codes = icx::kv_codes(G, BITS);
    const uint8_t* kd = c + (t16 * G + g) * 4 * BITS + i * BITS;
    const uint8_t* vd = c + codes + (((t16 >> 2) * 16 + 4 * i) * G + g) * BITS + (t16 & 3) * (BITS / 4);
    const float ks = icx::scale_of(c[icx::kv_key_scales(G, BITS) + t16 * G + g], 0);
    const float vs = icx::scale_of(c[icx::kv_value_scales(G, BITS) + ((t16 >> 2) * G + g) * 4 + (t16 & 3)], 0);
    if constexpr (BITS == 4) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(kd);
        unpack(icx::decode2<4, 0>(w, ks), k[0], k[1]);
        unpack(icx::decode2<4, 1>(w, ks), k[2], k[3]);
        unpack(icx::decode2<4, 2>(w, ks), k[4], k[5]);
        unpack(icx::decode2<4, 3>(w, ks), k[6], k[7]);
#pragma unroll
        for (int e = 0; e < 4; ++e) unpack(icx::decode2<4, 0>(vd[e * G * BITS], vs), v[e], v[4 + e]);
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(kd);
        unpack(icx::decode2<8, 0>(w.x, ks), k[0], k[1]);
        unpack(icx::decode2<8, 1>(w.x, ks), k[2], k[3]);
        unpack(icx::decode2<8, 0>(w.y, ks), k[4], k[5]);
        unpack(icx::decode2<8, 1>(w.y, ks), k[6], k[7]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            unpack(icx::decode2<8, 0>(*reinterpret_cast<const uint16_t*>(vd + e * G * BITS), vs), v[e], v[4 + e]);
    }
}

template <typename T>
__device__ __forceinline__ void put_values(const CacheArgs& a, int64_t t, int h, int G, int g, int i, const float (&k)[8],
                                           const float (&v)[8]) {
    const int64_t row = (t * a.l.heads + h) * (32 * (int64_t)G) + 32 * g;
    if (a.k_out) icx::store_f32(reinterpret_cast<T*>(a.k_out) + row + 8 * i, k);
    if (a.v_out) {
        float lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            lo[e] = v[e];
            hi[e] = v[4 + e];
        }
        T* vo = reinterpret_cast<T*>(a.v_out) + row + 4 * i;
        icx::store_f32(vo, lo);
        icx::store_f32(vo + 16, hi);
    }
}

template <int BITS, typename T>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(CacheArgs a) {
    const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t unit = id >> 2;
    const int i = (int)(id & 3);
    const int G = a.l.G;
    if (unit >= a.units) return;
    const int g = (int)(unit % G);
    const int64_t th = unit / G;
    const int h = (int)(th % a.l.heads);
    const int64_t t = th / a.l.heads;
    const int64_t slot = slot_of(a, t);
    float k[8], v[8];
    if (slot < 0 || slot >= a.slots_end) {
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = v[e] = 0.0f;
    } else {
        int t16;
        const uint8_t* c = chunk_of(a, slot, h, t16);
        take_codes<BITS>(c, G, t16, g, i, k, v);
    }
    put_values<T>(a, t, h, G, g, i, k, v);
}

// ---- 16 tokens and one head a wave ----------------------------------------------------------------
// The tokens 16 n - d .. + 15, d the place of the first slot in its chunk: a prompt that starts inside a chunk
// still meets the chunks after it from their start.
struct Sixteen {
    int64_t first;  // of the list; some may lie outside it
    int head;
    bool chunk;     // the slots are one chunk
    uint8_t* at;    // of that chunk
};

template <int W>
__device__ __forceinline__ Sixteen sixteen(const CacheArgs& a, int64_t (&slots)[W][16], int wid, int lane) {
    Sixteen s;
    const int64_t n = (int64_t)blockIdx.x * W + wid;
    s.head = (int)(n % a.l.heads);
    s.first = n / a.l.heads * 16 - (slot_of(a, 0) & 15);
    int64_t slot = -1;
    const int64_t t = s.first + (lane & 15);
    if (t >= 0 && t < a.tokens) slot = slot_of(a, t);
    if (slot >= a.slots_end) slot = -1;
    if (lane < 16) slots[wid][lane] = slot;
    const int lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)slot), hi = __builtin_amdgcn_readfirstlane((int)(slot >> 32));
    const int64_t base = (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
    s.chunk = __all(base >= 0 && (base & 15) == 0 && slot == base + (lane & 15));
    int t16;
    s.at = chunk_of(a, s.chunk ? base : 0, s.head, t16);
    __syncthreads();
    return s;
}

// Piece p of the wave's 64 G: block g of token t, lane i of its four.
template <int G>
__device__ __forceinline__ void piece(int p, int& t, int& g, int& i) {
    t = p / (4 * G);
    g = p % (4 * G) >> 2;
    i = p & 3;
}

template <int BITS, int G, typename T>
__global__ void __launch_bounds__(kThreads) kv_write_chunks_kernel(CacheArgs a) {
    constexpr int W = kThreads / 64, BYTES = 2 * (64 * G * BITS + 16 * G);
    __shared__ __attribute__((aligned(16))) uint8_t image[W][BYTES];
    __shared__ int64_t slots[W][16];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Sixteen s = sixteen<W>(a, slots, wid, lane);
    float k[G][8], v[G][8];
#pragma unroll
    for (int n = 0; n < G; ++n) {
        int t, g, i;
        piece<G>(n * 64 + lane, t, g, i);
        const int64_t tok = min(max(s.first + t, (int64_t)0), a.tokens - 1);
        icx::load_f32(reinterpret_cast<const T*>(a.k) + tok * a.k_token + s.head * a.k_head + 32 * g + 8 * i, k[n]);
        const T* vp = reinterpret_cast<const T*>(a.v) + tok * a.v_token + s.head * a.v_head + 32 * g + 4 * i;
        float lo[4], hi[4];
        icx::load_f32(vp, lo);
        icx::load_f32(vp + 16, hi);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[n][2 * e] = lo[e];
            v[n][2 * e + 1] = hi[e];
        }
    }
#pragma unroll
    for (int n = 0; n < G; ++n) {
        int t, g, i;
        piece<G>(n * 64 + lane, t, g, i);
        const uint32_t ke = icx::block_exponent<BITS>(block_top(k[n])), ve = icx::block_exponent<BITS>(block_top(v[n]));
        const uint2 kc = encode8<BITS>(k[n], ke), vc = encode8<BITS>(v[n], ve);
        uint8_t* c = image[wid];
        int t16 = t;
        if (!s.chunk) {
            const int64_t slot = slots[wid][t];
            if (slot < 0) continue;
            c = chunk_of(a, slot, s.head, t16);
        }
        put_codes<BITS>(c, G, t16, g, i, kc, vc, ke, ve);
    }
    __syncthreads();
    if (!s.chunk) return;
    const uint4* from = reinterpret_cast<const uint4*>(image[wid]);
    uint4* to = reinterpret_cast<uint4*>(s.at);
#pragma unroll
    for (int n = 0; n < (BYTES / 16 + 63) / 64; ++n)
        if (n * 64 + lane < BYTES / 16) to[n * 64 + lane] = from[n * 64 + lane];
}

// PAST: the cache is read past the GPU's own.
template <int BITS, int G, bool PAST, typename T>
__global__ void __launch_bounds__(kThreads) kv_read_chunks_kernel(CacheArgs a) {
    constexpr int W = kThreads / 64, BYTES = 2 * (64 * G * BITS + 16 * G);
    __shared__ __attribute__((aligned(16))) uint8_t image[W][BYTES];
    __shared__ int64_t slots[W][16];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Sixteen s = sixteen<W>(a, slots, wid, lane);
    if (s.chunk) {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        const u32x4* from = reinterpret_cast<const u32x4*>(s.at);
        u32x4* to = reinterpret_cast<u32x4*>(image[wid]);
#pragma unroll
        for (int n = 0; n < (BYTES / 16 + 63) / 64; ++n)
            if (n * 64 + lane < BYTES / 16) to[n * 64 + lane] = PAST ? __builtin_nontemporal_load(from + n * 64 + lane) : from[n * 64 + lane];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < G; ++n) {
        int t, g, i;
        piece<G>(n * 64 + lane, t, g, i);
        const int64_t tok = s.first + t;
        if (tok < 0 || tok >= a.tokens) continue;
        float k[8], v[8];
        if (s.chunk) {
            take_codes<BITS>(image[wid], G, t, g, i, k, v);
        } else {
            const int64_t slot = slots[wid][t];
            if (slot >= 0) {
                int t16;
                const uint8_t* c = chunk_of(a, slot, s.head, t16);
                take_codes<BITS>(c, G, t16, g, i, k, v);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) k[e] = v[e] = 0.0f;
            }
        }
        put_values<T>(a, tok, s.head, G, g, i, k, v);
    }
}

// What both entry points check, and the arguments they share.
int cache_args(const icx_kv_cache* c, const void* slots, int slots_dtype, size_t tokens, int dtype, const char* who,
               CacheArgs* a) {
    int rc = icx::check_kv_cache(c, who);
    if (rc) return rc;
    if (!icx::is_float_kind(dtype))
        ICX_FAIL(ICX_ERR_DTYPE, "%s: dtype %d unsupported (must be Float32, Float16 or BFloat16)", who, dtype);
    if (slots_dtype != ICX_I32 && slots_dtype != ICX_I64)
        ICX_FAIL(ICX_ERR_DTYPE, "%s: slots must be Int32 or Int64 (got dtype %d)", who, slots_dtype);
    *a = CacheArgs{};
    a->data = reinterpret_cast<uint8_t*>(c->data);
    a->l = icx::kv_layout(*c);
    a->page_size = c->page_size;
    a->slots_end = c->pages * c->page_size;
    a->slots = slots;
    a->slots64 = slots_dtype == ICX_I64;
    if (tokens > (size_t)INT64_MAX / 4 / ((size_t)c->kv_heads * (size_t)a->l.G))
        ICX_FAIL(ICX_ERR_SHAPE, "%s: %zu tokens are too many", who, tokens);
    a->tokens = (int64_t)tokens;
    a->units = a->tokens * c->kv_heads * a->l.G;
    // HIP's limit on the threads of a launch is 2^32 - 1
    if (a->units > (int64_t)0x3fffffff) ICX_FAIL(ICX_ERR_UNSUPPORTED, "%s: %zu tokens a call are too many", who, tokens);
    return ICX_OK;
}

// From how many heads of tokens on the kernels of 16 tokens a wave are taken.  8 heads of 128, 4 bits, us of
// either kernel: writes of 1024 tokens 3.9 / 4.4, of 2048 5.3 / 4.5, of 16384 19.7 / 13.3 (slots out of
// order 3.9 / 5.6, 5.4 / 6.1, 20.5 / 20.9); reads of 4096 6.3 / 6.8, of 16384 18.1 / 16.2, and of heads of
// 256 in float32 17.3 / 15.6 and 72.7 / 48.2.  12289 tokens of 12 heads of 64, 8 bits: written in 20.7 / 12.1,
// read in 15.2 / 11.6; 65536 of 8 heads of 128 read in 93 / 75 (5.4 TB/s).
constexpr int64_t kWriteByChunks = 16384, kReadByChunks = 32768;
unsigned chunk_blocks(const CacheArgs& a) {
    // (a group more for the tokens before the first whole one)
    return (unsigned)icx::cdiv((icx::cdiv((size_t)a.tokens, 16) + 1) * (size_t)a.l.heads, kThreads / 64);
}
template <int BITS, typename F>
void with_head(int G, F f) {
    std::integral_constant<int, BITS> bits;
    switch (G) {
        case 1: f(bits, std::integral_constant<int, 1>()); break;
        case 2: f(bits, std::integral_constant<int, 2>()); break;
        case 3: f(bits, std::integral_constant<int, 3>()); break;
        case 4: f(bits, std::integral_constant<int, 4>()); break;
        case 5: f(bits, std::integral_constant<int, 5>()); break;
        case 6: f(bits, std::integral_constant<int, 6>()); break;
        case 7: f(bits, std::integral_constant<int, 7>()); break;
        default: f(bits, std::integral_constant<int, 8>()); break;
    }
}
template <typename F>
void with_blocks(const icx::KvLayout& l, F f) {
    if (l.bits == 4) with_head<4>(l.G, f);
    else with_head<8>(l.G, f);
}

}  // namespace

int icx::check_kv_cache(const icx_kv_cache* c, const char* who) {
    if (!c || !c->data) ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: null cache", who);
    if (c->bits != 4 && c->bits != 8) ICX_FAIL(ICX_ERR_UNSUPPORTED, "%s: a cache has 4 or 8 bits (got %d)", who, c->bits);
    if (c->head_size < 32 || c->head_size > 256 || c->head_size % 32)
        ICX_FAIL(ICX_ERR_UNSUPPORTED, "%s: head size %d (must be a multiple of 32 up to 256)", who, c->head_size);
    if (c->page_size < 16 || c->page_size > 1024 || c->page_size % 16)
        ICX_FAIL(ICX_ERR_UNSUPPORTED, "%s: page size %d (must be a multiple of 16 up to 1024)", who, c->page_size);
    if (c->kv_heads < 1 || c->kv_heads > 1024 || c->pages < 1 || c->pages > 0x7fffffff)
        ICX_FAIL(ICX_ERR_SHAPE, "%s: %lld pages of %d heads", who, (long long)c->pages, c->kv_heads);
    if (reinterpret_cast<uintptr_t>(c->data) & 15)
        ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: the cache must be 16-byte aligned", who);
    return ICX_OK;
}

extern "C" size_t icx_kv_cache_bytes(const icx_kv_cache* c) {
    icx::clear_error();
    if (!c) return 0;
    icx_kv_cache d = *c;
    d.data = reinterpret_cast<void*>(16);  // a size is asked for before there is memory
    if (icx::check_kv_cache(&d, "KvCache")) return 0;
    return (size_t)d.pages * (size_t)icx::kv_layout(d).page_bytes;
}

extern "C" int icx_kv_cache_write(icx_stream_t stream, const icx_kv_cache* cache, const icx_kv_write* args) {
    icx::clear_error();
    const char* who = "KvCacheWrite";
    if (!args) ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: null arguments", who);
    CacheArgs a;
    int rc = cache_args(cache, args->slots, args->slots_dtype, args->tokens, args->dtype, who, &a);
    if (rc) return rc;
    if (args->tokens == 0) return ICX_OK;
    if (!args->k || !args->v || !args->slots) ICX_FAIL(ICX_ERR_INVALID_ARG, "%s: null k, v or slots", who);
    a.k = args->k;
    a.v = args->v;
    a.k_token = args->k_token_stride;
    a.k_head = args->k_head_stride;
    a.v_token = args->v_token_stride;
    a.v_head = args->v_head_stride;
    const unsigned blocks = (unsigned)icx::cdiv((size_t)a.units * 4, kThreads);
    return icx::with_float_type(args->dtype, [&](auto* t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        if (a.tokens * a.l.heads >= kWriteByChunks) 
            with_blocks(a.l, [&](auto bits, auto g) {
                constexpr int B = decltype(bits)::value, G = decltype(g)::value;
                kv_write_chunks_kernel<B, G, T><<<chunk_blocks(a), kThreads, 0, (hipStream_t)stream>>>(a);
            });
        else if (cache->bits == 4) kv_write_kernel<4, T><<<blocks, kThreads, 0, (hipStream_t)stream>>>(a);
        else kv_write_kernel<8, T><<<blocks, kThreads, 0, (hipStream_t)stream>>>(a);
        ICX_LAUNCH_CHECK("kv_write_kernel");
        return ICX_OK;
    });
}

extern "C" int icx_kv_cache_read(icx_stream_t stream, const icx_kv_cache* cache, const void* slots, int slots_dtype,
                                 size_t tokens, void* k, void* v, int dtype) {
    icx::clear_error();
    CacheArgs a;
    int rc = cache_args(cache, slots, slots_dtype, tokens, dtype, "KvCacheRead", &a);
    if (rc) return rc;
    if (tokens == 0 || (!k && !v)) return ICX_OK;
    if (!slots) ICX_FAIL(ICX_ERR_INVALID_ARG, "KvCacheRead: null slots");
    // What moves more than the last-level cache's 256 MB would put its own codes out before they were read again (65536
    // tokens of 8 heads of 128 in 8 bits 78.7 us for 82.8; 12289 of 12 of 64, just written, 13.3 for 12.9 so: left).
    const int64_t block_bytes = 2 * (4 * (int64_t)cache->bits + 1 + 32 * (dtype == ICX_F32 ? 4 : 2));
    const bool past = a.units * block_bytes > ((int64_t)1 << 28);
    a.k_out = k;
    a.v_out = v;
    const unsigned blocks = (unsigned)icx::cdiv((size_t)a.units * 4, kThreads);
    return icx::with_float_type(dtype, [&](auto* t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        if (a.tokens * a.l.heads >= kReadByChunks) 
            with_blocks(a.l, [&](auto bits, auto g) {
                constexpr int B = decltype(bits)::value, G = decltype(g)::value;
                if (past) kv_read_chunks_kernel<B, G, true, T><<<chunk_blocks(a), kThreads, 0, (hipStream_t)stream>>>(a);
                else kv_read_chunks_kernel<B, G, false, T><<<chunk_blocks(a), kThreads, 0, (hipStream_t)stream>>>(a);
            });
        else if (cache->bits == 4) kv_read_kernel<4, T><<<blocks, kThreads, 0, (hipStream_t)stream>>>(a);
        else kv_read_kernel<8, T><<<blocks, kThreads, 0, (hipStream_t)stream>>>(a);
        ICX_LAUNCH_CHECK("kv_read_kernel");
        return ICX_OK;
    });
}
