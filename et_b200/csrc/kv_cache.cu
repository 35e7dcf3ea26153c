// A cache of keys and values in int8, in pages: rows of K and V quantised as they are written (a scale for each row and head: its largest size / 127), and rows read back.
//
// codes [pages][K, V][heads][page rows][head_dim], scales [pages][K, V][heads][page rows]: a page of a head is one piece. Neighbouring lanes have a
// row of a head, 16 features each: 16 bytes of codes, 32 of fp16. Heads of a token lie side by side in a block, whose threads take the same row of several tokens at once. Bound by memory: 3 bytes a feature.
#include <algorithm>
#include "common.h"
#include "ptx.cuh"
#include "vec_math.cuh"

namespace et {
namespace {

// 27 thousand rows of 16 heads of 128 read back, with one, two, four, eight tokens of a thread in flight: 31.7, 28.3, 38.7, 46.5 us, written (8192 tokens) 13.9, 13.3,
// 13.5, 17.4, blocks of 256 threads 30.3 and 13.3; few tokens with one and two 2.25 and 2.86.
constexpr int kThreads = 128;
constexpr int kBlockRows = 4;    // of a token, at most, in a block

struct CacheParams {
    int8_t* codes;
    float* scales;
    half *k, *v;                 // read by the write, written by the read
    const int* slots;
    long long k_pitch, v_pitch, n_slots;
    int tokens, heads, head_dim, page;
    int lanes;                   // of a row, a power of two
    int block_rows, block_tokens;   // rows of a token, and tokens, side by side in a block
};

// What a thread works on: 16 features of row (side, head) of tokens first, first + step, ..
struct CachePlace {
    bool in;
    int at, row, first, step;
};
__device__ __forceinline__ CachePlace cache_place(const CacheParams& p, int tokens) {
    const int g = threadIdx.x / p.lanes, t = g / p.block_rows;
    CachePlace c;
    c.at = (threadIdx.x & (p.lanes - 1)) * 16;
    c.row = blockIdx.y * p.block_rows + g - t * p.block_rows;
    c.first = blockIdx.x * (p.block_tokens * tokens) + t;
    c.step = p.block_tokens;
    c.in = t < p.block_tokens && c.row < 2 * p.heads;
    return c;
}
// Where a token's row lies among the cache's rows; below 0: no place.
__device__ __forceinline__ long long cache_row(const CacheParams& p, int token, int row) {
    const int slot = p.slots[token], page = slot / p.page;
    return slot < 0 || slot >= p.n_slots ? -1 : ((long long)page * (2 * p.heads) + row) * p.page + (slot - page * p.page);
}
__device__ __forceinline__ half* token_row(const CacheParams& p, int token, int row) {
    return row >= p.heads ? p.v + token * p.v_pitch + (row - p.heads) * p.head_dim : p.k + token * p.k_pitch + row * p.head_dim;
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

// code = x / scale to the nearest, of two equally near the even one; x / scale is corrected by what its product with the scale leaves, so that it is the
// rounded quotient. The code comes out of the low bits of 1.5 2^23 + x / scale, to which the addition rounds it.
// kTokens: of a thread, all requested at once.
template <bool kVec, int kTokens>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const __grid_constant__ CacheParams p) {
    const CachePlace c = cache_place(p, kTokens);
    const bool features = c.at < p.head_dim;
    pdl_wait();
    pdl_launch_dependents();
    uint4 x[kTokens][2];
    long long to[kTokens];
#pragma unroll
    for (int n = 0; n < kTokens; ++n) {
        const int token = c.first + n * c.step;
        x[n][0] = x[n][1] = make_uint4(0u, 0u, 0u, 0u);
        to[n] = -1;
        if (c.in && token < p.tokens) {
            to[n] = cache_row(p, token, c.row);
            if (features) {   // (read whether it has a place or not: both are on their way at once)
                const half* const from = token_row(p, token, c.row) + c.at;
                x[n][0] = load8<kVec>(from);
                x[n][1] = load8<kVec>(from + 8);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < kTokens; ++n) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 v = __half22float2(reinterpret_cast<const half2*>(x[n])[i]);
            top = max_nan(top, max_nan(fabsf(v.x), fabsf(v.y)));
        }
        for (int o = p.lanes >> 1; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (to[n] < 0) continue;
        const float scale = top / 127.f, inverse = scale > 0.f ? 1.f / scale : 0.f;
        if (features) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t b[4];
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    const float2 v = __half22float2(reinterpret_cast<const half2*>(x[n])[i * 2 + k / 2]);
                    const float q0 = v.x * inverse, q1 = v.y * inverse;
                    const float r0 = fmaf(fmaf(-q0, scale, v.x), inverse, q0), r1 = fmaf(fmaf(-q1, scale, v.y), inverse, q1);
                    b[k] = __float_as_uint(r0 + 12582912.f);
                    b[k + 1] = __float_as_uint(r1 + 12582912.f);
                }
                w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            }
            *reinterpret_cast<uint4*>(p.codes + to[n] * p.head_dim + c.at) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (c.at == 0) p.scales[to[n]] = scale - scale == 0.f ? scale : __int_as_float(0x7fffffff);   // (infinite: all of the row is not a number)
    }
}

template <bool kVec, int kTokens>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const __grid_constant__ CacheParams p) {
    const CachePlace c = cache_place(p, kTokens);
    if (!c.in || c.at >= p.head_dim) return;
    pdl_wait();
    pdl_launch_dependents();
    uint4 w[kTokens];
    float scale[kTokens];
    bool there[kTokens];
#pragma unroll
    for (int n = 0; n < kTokens; ++n) {
        const int token = c.first + n * c.step;
        const long long row = token < p.tokens ? cache_row(p, token, c.row) : -1;
        there[n] = row >= 0;
        if (there[n]) {
            w[n] = *reinterpret_cast<const uint4*>(p.codes + row * p.head_dim + c.at);
            scale[n] = p.scales[row];
        }
    }
#pragma unroll
    for (int n = 0; n < kTokens; ++n) {
        if (!there[n]) continue;
        const uint32_t u[4] = {w[n].x ^ 0x80808080u, w[n].y ^ 0x80808080u, w[n].z ^ 0x80808080u, w[n].w ^ 0x80808080u};
        uint4 v[2];
        half2* const h = reinterpret_cast<half2*>(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {   // the byte + 128 as the low bits of 2^23
            const float lo = __uint_as_float(__byte_perm(u[i / 2], 0x4b000000u, i & 1 ? 0x7442 : 0x7440)) - 8388736.f;
            const float hi = __uint_as_float(__byte_perm(u[i / 2], 0x4b000000u, i & 1 ? 0x7443 : 0x7441)) - 8388736.f;
            h[i] = __floats2half2_rn(lo * scale[n], hi * scale[n]);
        }
        half* const to = token_row(p, c.first + n * c.step, c.row) + c.at;
        store8<kVec>(to, v[0]);
        store8<kVec>(to + 8, v[1]);
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
    if (a->tokens > 0x7ff00000) return bad("too many rows");
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
    p.tokens = a->tokens; p.heads = a->heads; p.head_dim = a->head_dim; p.page = a->page;
    const bool vec = aligned16(a->k) && aligned16(a->v) && (a->tokens == 1 || ((a->k_pitch | a->v_pitch) & 7) == 0);
    p.lanes = 1;
    while (p.lanes * 16 < a->head_dim) p.lanes *= 2;
    const int groups = kThreads / p.lanes, rows = 2 * a->heads;
    p.block_rows = std::min(std::min(groups, rows), kBlockRows);
    p.block_tokens = groups / p.block_rows;
    // Two tokens to a thread where that leaves the SMs their blocks.
    const unsigned grid_y = (unsigned)((rows + p.block_rows - 1) / p.block_rows);
    const long long blocks = (a->tokens + (long long)p.block_tokens - 1) / p.block_tokens;
    const int in_flight = blocks * grid_y >= 16LL * sm_count() ? 2 : 1;
    const dim3 grid((unsigned)((blocks + in_flight - 1) / in_flight), grid_y);
    static void (*const kernels[2][2][2])(CacheParams) = {{{cache_read_kernel<false, 1>, cache_read_kernel<false, 2>}, {cache_read_kernel<true, 1>, cache_read_kernel<true, 2>}},
                                                          {{cache_write_kernel<false, 1>, cache_write_kernel<false, 2>}, {cache_write_kernel<true, 1>, cache_write_kernel<true, 2>}}};
    const auto kernel = kernels[write][vec][in_flight - 1];
    return cuda_status(launch_pdl(kernel, grid, dim3(kThreads), 0, static_cast<cudaStream_t>(a->stream), p), where);
}

}  // namespace
}  // namespace et

extern "C" int et_kv_cache_write(const et_kv_cache_args* a) { return et::cache_run(a, true, "et_kv_cache_write"); }
extern "C" int et_kv_cache_read(const et_kv_cache_args* a) { return et::cache_run(a, false, "et_kv_cache_read"); }
