// Attention of drafted tokens over a cache of int8 codes: what its kernels share.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <climits>
#include <cstdint>
#include "vec_math.cuh"

namespace et {

struct TreeParams {
    half* out;
    const half* q;
    const int8_t* codes;                   // [pages][K, V][K/V heads][page][head_dim]
    const float* scales;                   // [pages][K, V][K/V heads][page]
    const int *table, *k_lens, *cu_seqlens;
    const long long* tree;                 // bits of the drafted tokens that each one sees, or null: those up to itself
    long long out_pitch, q_pitch;
    int nhead, group, head_dim;            // group: query heads to a K/V head
    int batch, q_tokens, max_q_len, max_k_len;
    int pages, page, table_width;
    float scale_log2;                      // q . k -> log2 domain
};

// Where a sequence's drafted tokens and keys are.
struct TreeSeq {
    int q0, qlen, klen;
    int kept;                              // keys before the drafted ones (below 0: there are fewer keys than tokens)
};

// The b-th sequence in order of length (the one that has b longer, or as long and earlier, ones) becomes b; its keys. By a block of at least as many threads as there are sequences.
template <int kThreads>
__device__ __forceinline__ int nth_longest(const TreeParams& p, int& b) {
    __shared__ __align__(16) int lens[kThreads];
    __shared__ int found[2];
    const int i = threadIdx.x, len = i < p.batch ? p.k_lens[i] : INT_MIN;
    lens[i] = len;
    __syncthreads();
    if (i < p.batch) {
        int before = 0;
        for (int j = 0; j < p.batch; j += 4) {
            const int4 l = *reinterpret_cast<const int4*>(lens + j);
            before += (l.x > len || (l.x == len && j < i)) + (l.y > len || (l.y == len && j + 1 < i)) + (l.z > len || (l.z == len && j + 2 < i)) + (l.w > len || (l.w == len && j + 3 < i));
        }
        if (before == b) {
            found[0] = i;
            found[1] = len;
        }
    }
    __syncthreads();
    b = found[0];
    return found[1];
}

// keys: k_lens[b]
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int b, int keys) {
    TreeSeq s;
    if (p.cu_seqlens) {
        s.q0 = p.cu_seqlens[b];
        s.qlen = p.cu_seqlens[b + 1] - s.q0;
    } else {
        s.q0 = b * p.max_q_len;
        s.qlen = p.max_q_len;
    }
    s.qlen = s.q0 < 0 ? 0 : max(0, min(s.qlen, min(p.max_q_len, p.q_tokens - s.q0)));
    const int len = max(0, keys);
    s.kept = len - s.qlen;
    s.klen = (int)min((long long)min(len, p.max_k_len), (long long)p.table_width * p.page);
    return s;
}
// The bits of drafted token i of a sequence.
__device__ __forceinline__ unsigned long long tree_bits(const TreeParams& p, const TreeSeq& s, int i) {
    return p.tree ? (unsigned long long)p.tree[s.q0 + i] : (2ull << i) - 1ull;
}
__device__ __forceinline__ bool tree_sees(const TreeSeq& s, unsigned long long bits, int key) {
    const int place = key - s.kept;
    return key < s.klen && (place < 0 || (place < 64 && ((bits >> place) & 1ull)));
}

// 16 keys of a head in a page, as far as a panel has their features, of K and of V.
__device__ __forceinline__ void load_keys(uint32_t to, const void* tmap, int feature, int row, int head, int page_side, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to), "l"(tmap), "r"(feature), "r"(row), "r"(head),
                 "r"(page_side), "r"(bar)
                 : "memory");
}
template <int kSize>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
    if constexpr (kSize == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(kSize) : "memory");
}

// Codes become halves without a conversion: the byte + 128 as the low bits of 1024 is 1024 + byte + 128 in fp16, exactly, from which 1152 is taken.
__device__ __forceinline__ uint32_t codes_biased(uint32_t four) { return four ^ 0x80808080u; }
template <int kHigh>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t biased) {   // bytes 0 and 1, or 2 and 3
    const uint32_t v = __byte_perm(biased, 0x64646464u, kHigh ? 0x4342 : 0x4140);
    const half2 h = __hsub2(*reinterpret_cast<const half2*>(&v), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Values scales enter the weights of the second product (as codes are whole numbers there), which are fp16. So the reference that is taken from a row's scores follows
// score + log2 of the value's scale, in steps of kRescaleStep, and the weights are 2^kLift times as large: the largest weight times its scale lies between 2^7 and 2^15, and one that falls below half of
// fp16's smallest step is below 2^-32 of it. (Without the lift below 2^-25: of 60000 keys with such weights nothing was left, even in features where the large one's value is 0.) This is that logarithm; scales
// below 2^-40 (rows of zeros: the smallest others are 2^-31) count as 2^-40.
constexpr float kRescaleStep = 8.f, kLift = 7.f;   // log2 units
__device__ __forceinline__ float log2_of_scale(float s) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaxf(s, 9.094947017729282e-13f)));
    return y;
}

// A part of a row's sums counts if it has a reference (its scores may not be numbers: it is given one then); a part without one has seen nothing.
__device__ __forceinline__ bool tree_saw(float reference) { return reference != -INFINITY; }

}  // namespace et
