// Writing keys and values into the quantized cache and reading them back (kv_format.hpp has the
// format).
//
// Four lanes share a block of 32 values.  A lane takes 8 consecutive keys (its codes are then a
// whole dword or two of the token's row), and of the values 4 consecutive ones of each half of the
// block, the pairs that a byte of the transposed layout holds.  Both kernels are bound by memory;
// the conversions are one instruction a pair.
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
    const int codes = icx::kv_codes(G, BITS);
    uint8_t* kd = c + (t16 * G + g) * 4 * BITS + i * BITS;
    if (BITS == 4) *reinterpret_cast<uint32_t*>(kd) = kc.x;
    else *reinterpret_cast<uint2*>(kd) = kc;
    uint8_t* vd = c + codes + (((t16 >> 2) * 16 + 4 * i) * G + g) * BITS + (t16 & 3) * (BITS / 4);
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

__device__ __forceinline__ void unpack(uint32_t w, float& lo, float& hi) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
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
        if (cache->bits == 4) kv_write_kernel<4, T><<<blocks, kThreads, 0, (hipStream_t)stream>>>(a);
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
    a.k_out = k;
    a.v_out = v;
    const unsigned blocks = (unsigned)icx::cdiv((size_t)a.units * 4, kThreads);
    return icx::with_float_type(dtype, [&](auto* t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        if (cache->bits == 4) kv_read_kernel<4, T><<<blocks, kThreads, 0, (hipStream_t)stream>>>(a);
        else kv_read_kernel<8, T><<<blocks, kThreads, 0, (hipStream_t)stream>>>(a);
        ICX_LAUNCH_CHECK("kv_read_kernel");
        return ICX_OK;
    });
}
