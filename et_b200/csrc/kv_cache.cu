// A cache of keys and values in int8, in pages: rows of K and V quantised as they are written (a scale for each row and head: its largest size / 127), and rows read back.
//
// codes [pages][K, V][heads][page rows][head_dim], scales [pages][K, V][heads][page rows]: a page of a head is one piece. A group of neighbouring lanes has a
// row of a head, 8 features to a lane, so that fp16 rows go as 16 bytes a lane and codes as 8; heads of a token lie side by side in a warp. Bound by memory: 3 bytes a feature.
#include "common.h"
#include "ptx.cuh"
#include "vec_math.cuh"

namespace et {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsInFlight = 4;

struct CacheParams {
    int8_t* codes;
    float* scales;
    half *k, *v;                 // read by the write, written by the read
    const int* slots;
    long long k_pitch, v_pitch, n_slots;
    long long items;             // tokens x K, V x heads
    int heads, head_dim, page;
};

// Row (token, side, head) with number i, in which heads of a token's K and then of its V are neighbours.
struct CacheRow {
    half* x;
    long long at;                // among the cache's rows; below 0: no place
};
__device__ __forceinline__ CacheRow cache_row(const CacheParams& p, long long i) {
    const int per_token = 2 * p.heads;
    const long long token = i / per_token;
    const int r = (int)(i - token * per_token), side = r >= p.heads, head = r - side * p.heads;
    const int slot = p.slots[token];
    CacheRow c;
    c.x = (side ? p.v + token * p.v_pitch : p.k + token * p.k_pitch) + head * p.head_dim;
    const int page = slot / p.page;
    c.at = slot < 0 || slot >= p.n_slots ? -1 : ((long long)page * per_token + r) * p.page + (slot - page * p.page);
    return c;
}

// fp16 rows in whole 16 bytes, or elements one by one.
template <bool kVec>
__device__ __forceinline__ uint4 load8(const half* x) {
    if constexpr (kVec) return *reinterpret_cast<const uint4*>(x);
    uint4 v;
    half* const h = reinterpret_cast<half*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = x[i];
    return v;
}
template <bool kVec>
__device__ __forceinline__ void store8(half* x, const uint4& v) {
    if constexpr (kVec) {
        *reinterpret_cast<uint4*>(x) = v;
    } else {
        const half* const h = reinterpret_cast<const half*>(&v);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = h[i];
    }
}

// lanes: of a group, a power of two. code = x / scale to the nearest, of two equally near the even one; x / scale is corrected by what its product with the scale
// leaves, so that it is the rounded quotient.
template <bool kVec>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const __grid_constant__ CacheParams p, int lanes) {
    const int at = (threadIdx.x & (lanes - 1)) * 8, groups = kThreads / lanes;
    const long long first = (long long)blockIdx.x * groups * kRowsInFlight + threadIdx.x / lanes;
    pdl_wait();
    pdl_launch_dependents();
    uint4 x[kRowsInFlight];
    long long to[kRowsInFlight];
#pragma unroll
    for (int n = 0; n < kRowsInFlight; ++n) {
        const long long i = first + n * groups;
        x[n] = make_uint4(0u, 0u, 0u, 0u);
        to[n] = -1;
        if (i < p.items) {
            const CacheRow c = cache_row(p, i);
            to[n] = c.at;
            if (c.at >= 0 && at < p.head_dim) x[n] = load8<kVec>(c.x + at);
        }
    }
#pragma unroll
    for (int n = 0; n < kRowsInFlight; ++n) {
        float f[8], top = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = __half22float2(reinterpret_cast<const half2*>(&x[n])[i]);
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
            top = max_nan(top, max_nan(fabsf(v.x), fabsf(v.y)));
        }
        for (int o = lanes >> 1; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (to[n] < 0) continue;
        const float scale = top / 127.f, inverse = scale > 0.f ? 1.f / scale : 0.f;
        if (at < p.head_dim) {
            uint32_t w[2] = {0u, 0u};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float q = f[i] * inverse;
                w[i >> 2] |= (uint32_t)(uint8_t)(int8_t)__float2int_rn(fmaf(fmaf(-q, scale, f[i]), inverse, q)) << (8 * (i & 3));
            }
            *reinterpret_cast<uint2*>(p.codes + to[n] * p.head_dim + at) = make_uint2(w[0], w[1]);
        }
        if (at == 0) p.scales[to[n]] = scale;
    }
}

template <bool kVec>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const __grid_constant__ CacheParams p, int lanes) {
    const int at = (threadIdx.x & (lanes - 1)) * 8, groups = kThreads / lanes;
    const long long first = (long long)blockIdx.x * groups * kRowsInFlight + threadIdx.x / lanes;
    pdl_wait();
    pdl_launch_dependents();
    uint2 c[kRowsInFlight];
    float scale[kRowsInFlight];
    half* to[kRowsInFlight];
#pragma unroll
    for (int n = 0; n < kRowsInFlight; ++n) {
        const long long i = first + n * groups;
        to[n] = nullptr;
        if (i < p.items && at < p.head_dim) {
            const CacheRow r = cache_row(p, i);
            if (r.at >= 0) {
                to[n] = r.x + at;
                c[n] = *reinterpret_cast<const uint2*>(p.codes + r.at * p.head_dim + at);
                scale[n] = p.scales[r.at];
            }
        }
    }
#pragma unroll
    for (int n = 0; n < kRowsInFlight; ++n) {
        if (!to[n]) continue;
        uint4 v;
        half2* const h = reinterpret_cast<half2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = (i < 2 ? c[n].x : c[n].y) >> (16 * (i & 1));
            h[i] = __floats2half2_rn((float)(int8_t)w * scale[n], (float)(int8_t)(w >> 8) * scale[n]);
        }
        store8<kVec>(to[n], v);
    }
}

int cache_run(const et_kv_cache_args* a, bool write, const char* where) {
    char text[96];
    auto bad = [&](const char* what) {
        std::snprintf(text, sizeof(text), "%s: %s", where, what);
        return fail(ET_ERR_INVALID, text);
    };
    if (!a) return bad("null pointer");
    if (a->tokens < 0 || a->pages < 0) return bad("negative size");
    if (a->heads < 1 || a->heads > 65535) return bad("heads must be 1 to 65535");
    if (a->head_dim < 16 || a->head_dim > 256 || a->head_dim % 16) return bad("head_dim must be a multiple of 16 up to 256");
    if (a->page < 16 || a->page % 16) return bad("the rows of a page must be a multiple of 16");
    if ((long long)a->pages * a->page > 0x7fffffff) return bad("more places than 32 bits number");
    if (a->tokens == 0) return ET_OK;
    if (!a->codes || !a->scales || !a->k || !a->v || !a->slots) return bad("null pointer");
    if (!aligned16(a->codes)) return bad("codes must start on 16 bytes");
    const long long width = (long long)a->heads * a->head_dim;
    if (a->tokens > 1 && (a->k_pitch < width || a->v_pitch < width)) return bad("pitch below the width of the heads");
    CacheParams p;
    p.codes = static_cast<int8_t*>(a->codes); p.scales = a->scales;
    p.k = static_cast<half*>(a->k); p.v = static_cast<half*>(a->v); p.slots = a->slots;
    p.k_pitch = a->k_pitch; p.v_pitch = a->v_pitch; p.n_slots = (long long)a->pages * a->page;
    p.items = (long long)a->tokens * 2 * a->heads;
    p.heads = a->heads; p.head_dim = a->head_dim; p.page = a->page;
    const bool vec = aligned16(a->k) && aligned16(a->v) && (a->tokens == 1 || ((a->k_pitch | a->v_pitch) & 7) == 0);
    int lanes = 2;
    while (lanes * 8 < a->head_dim) lanes *= 2;
    const long long rows = (long long)kThreads / lanes * kRowsInFlight, blocks = (p.items + rows - 1) / rows;
    if (blocks > 0x7fffffff) return bad("too many rows");
    const auto kernel = write ? (vec ? cache_write_kernel<true> : cache_write_kernel<false>) : (vec ? cache_read_kernel<true> : cache_read_kernel<false>);
    return cuda_status(launch_pdl(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, static_cast<cudaStream_t>(a->stream), p, lanes), where);
}

}  // namespace
}  // namespace et

extern "C" int et_kv_cache_write(const et_kv_cache_args* a) { return et::cache_run(a, true, "et_kv_cache_write"); }
extern "C" int et_kv_cache_read(const et_kv_cache_args* a) { return et::cache_run(a, false, "et_kv_cache_read"); }
