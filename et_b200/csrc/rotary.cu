// Rotary positions over several axes: the features of every head of Q and K are turned in pairs, pair i of a token by
//   angle = positions[token][axis[i]] * inv_freq[i],   (x, y) -> (x cos - y sin, x sin + y cos),
// x and y being features i and i + rot / 2 of the head, or 2i and 2i + 1; features from rot on are passed on as they are.
//
// What bounds it: HBM, each head is read and written once. The angle is taken in 64 bits: of a position of a million an fp32 product keeps
// four digits behind the point. In turns (multiplied by 1 / 2 pi) it loses its whole part there, and sine and cosine of the rest are fp32
// (sincospif). A block requests its heads, 16 bytes and four heads to a thread, takes the angles of its tokens meanwhile, once for all heads, and leaves
// them in shared memory; a thread keeps the eight that it needs in registers. 32768 tokens of 32 heads of 64 take 41 us, 6.5 TB/s; with the heads requested
// behind the angles and a warp's rows in different tokens 56. 5003 tokens of 40 heads of 128, neighbours, 96 features turned: 18 us, 5.6 TB/s.
#include "common.h"

namespace et {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kHeadsInFlight = 4;

enum Pairing {
    kHalves8 = 0,      // pairs half a rotated width apart, that half a multiple of 8: a thread has eight pairs, two granules of 16 bytes
    kHalves = 1,       // the same for any half: a thread has a granule and fetches the partners of its features, which straddle two others
    kNeighbours = 2,   // pairs of neighbouring features: a granule has its own partners, a thread four pairs
    kScalar = 3,       // anything else (heads or rows that do not start on 16 bytes): a thread has one pair
};

struct RotaryParams {
    half *q_out, *k_out;
    const half *q, *k;
    long long q_out_pitch, q_pitch, k_out_pitch, k_pitch;
    const int* positions;
    const float* inv_freq;
    const int* axis;
    int nhead_q, nhead_k, head_dim, rot, n_axes, tokens;
    int lanes;            // threads to a head (kHalves: a power of two, so that a head lies inside a warp)
    int block_tokens, head_step;   // tokens of a block, heads of each that it takes at a time
    bool interleaved;
    bool in_place_q, in_place_k;
};

// Eight fp16 values and back, products in fp32.
__device__ __forceinline__ void unpack8(const uint4& g, float (&v)[8]) {
    const half2* h = reinterpret_cast<const half2*>(&g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    uint4 g;
    half2* h = reinterpret_cast<half2*>(&g);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    return g;
}

template <int kPairing>
__global__ void __launch_bounds__(kMaxThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
    extern __shared__ float2 turns[];   // [block_tokens][rot / 2]: cosine, sine
    const int pairs = p.rot >> 1, heads = p.nhead_q + p.nhead_k;
    const int t0 = blockIdx.x * p.block_tokens, nt = min(p.block_tokens, p.tokens - t0);
    pdl_launch_dependents();
    pdl_wait();
    const int row = threadIdx.x / p.lanes, lane = threadIdx.x % p.lanes;   // (neighbouring heads of a token lie side by side)
    const int head_step = p.head_step, t = row / head_step, first_head = row % head_step;
    const bool token_in = t < nt;
    const float2* const cs = turns + min(t, nt - 1) * pairs;
    const long long q_row = (t0 + t) * p.q_pitch, k_row = (t0 + t) * p.k_pitch - p.nhead_q * p.head_dim;
    const long long q_out_row = (t0 + t) * p.q_out_pitch, k_out_row = (t0 + t) * p.k_out_pitch - p.nhead_q * p.head_dim;
    auto src = [&](int h) { return (h < p.nhead_q ? p.q + q_row : p.k + k_row) + h * p.head_dim; };
    auto dst = [&](int h) { return (h < p.nhead_q ? p.q_out + q_out_row : p.k_out + k_out_row) + h * p.head_dim; };
    auto in_place = [&](int h) { return h < p.nhead_q ? p.in_place_q : p.in_place_k; };
    // The block's angles, into shared memory. Called when the first heads are already on their way.
    auto take_angles = [&]() {
        for (int i = threadIdx.x; i < nt * pairs; i += blockDim.x) {
            const int pair = i % pairs;
            const int ax = p.axis[pair];
            float2 v = make_float2(1.f, 0.f);
            if (ax >= 0 && ax < p.n_axes) {   // (a pair of no axis is not turned)
                double turn = (double)p.positions[(size_t)(t0 + i / pairs) * p.n_axes + ax] * (double)p.inv_freq[pair] * 0.15915494309189535;
                turn -= rint(turn);
                sincospif(2.f * (float)turn, &v.y, &v.x);
            }
            turns[i] = v;
        }
        __syncthreads();
    };

    if constexpr (kPairing == kScalar) {
        take_angles();
        if (!token_in) return;
        for (int h = first_head; h < heads; h += head_step) {
            const half* const x = src(h);
            half* const y = dst(h);
            for (int i = lane; i < pairs; i += p.lanes) {
                const int a = p.interleaved ? 2 * i : i, b = p.interleaved ? 2 * i + 1 : i + pairs;
                const float u = __half2float(x[a]), v = __half2float(x[b]);
                y[a] = __float2half_rn(u * cs[i].x - v * cs[i].y);
                y[b] = __float2half_rn(u * cs[i].y + v * cs[i].x);
            }
            if (!in_place(h))
                for (int i = p.rot + lane; i < p.head_dim; i += p.lanes) y[i] = x[i];
        }
    } else if constexpr (kPairing == kHalves8) {
        const int turned = pairs / 8;   // lanes below have eight pairs, the others a granule that is passed on
        const bool turns_it = lane < turned;
        const int at = turns_it ? lane * 8 : p.rot + (lane - turned) * 8;
        const bool in = token_in && at < p.head_dim;
        uint4 a[kHeadsInFlight], b[kHeadsInFlight];
        auto fetch = [&](int h0) {
#pragma unroll
            for (int k = 0; k < kHeadsInFlight; ++k) {
                const int h = h0 + k * head_step;
                if (!in || h >= heads || (!turns_it && in_place(h))) continue;
                a[k] = *reinterpret_cast<const uint4*>(src(h) + at);
                if (turns_it) b[k] = *reinterpret_cast<const uint4*>(src(h) + at + pairs);
            }
        };
        fetch(first_head);
        take_angles();
        if (!in) return;
        float c[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 v = cs[turns_it ? at + i : 0];
            c[i] = v.x;
            s[i] = v.y;
        }
        for (int h0 = first_head; h0 < heads; h0 += head_step * kHeadsInFlight) {
            if (h0 != first_head) fetch(h0);
#pragma unroll
            for (int k = 0; k < kHeadsInFlight; ++k) {
                const int h = h0 + k * head_step;
                if (h >= heads || (!turns_it && in_place(h))) continue;
                half* const y = dst(h) + at;
                if (turns_it) {
                    half2 *const u = reinterpret_cast<half2*>(&a[k]), *const v = reinterpret_cast<half2*>(&b[k]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 x = __half22float2(u[i]), z = __half22float2(v[i]);
                        u[i] = __floats2half2_rn(x.x * c[2 * i] - z.x * s[2 * i], x.y * c[2 * i + 1] - z.y * s[2 * i + 1]);
                        v[i] = __floats2half2_rn(x.x * s[2 * i] + z.x * c[2 * i], x.y * s[2 * i + 1] + z.y * c[2 * i + 1]);
                    }
                    *reinterpret_cast<uint4*>(y + pairs) = b[k];
                }
                *reinterpret_cast<uint4*>(y) = a[k];
            }
        }
    } else if constexpr (kPairing == kNeighbours) {
        const int at = lane * 8, n_turned = max(0, min(4, (p.rot - at) / 2));   // pairs of the granule that are turned; the others are passed on
        const bool in = token_in && at < p.head_dim && (n_turned > 0 || !(p.in_place_q && p.in_place_k));
        uint4 a[kHeadsInFlight];
        auto fetch = [&](int h0) {
#pragma unroll
            for (int k = 0; k < kHeadsInFlight; ++k) {
                const int h = h0 + k * head_step;
                if (in && h < heads) a[k] = *reinterpret_cast<const uint4*>(src(h) + at);
            }
        };
        fetch(first_head);
        take_angles();
        if (!in) return;
        float2 turn[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) turn[i] = i < n_turned ? cs[at / 2 + i] : make_float2(1.f, 0.f);
        for (int h0 = first_head; h0 < heads; h0 += head_step * kHeadsInFlight) {
            if (h0 != first_head) fetch(h0);
#pragma unroll
            for (int k = 0; k < kHeadsInFlight; ++k) {
                const int h = h0 + k * head_step;
                if (h >= heads) continue;
                half2* const x = reinterpret_cast<half2*>(&a[k]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 v = __half22float2(x[i]);
                    const half2 z = __floats2half2_rn(v.x * turn[i].x - v.y * turn[i].y, v.x * turn[i].y + v.y * turn[i].x);
                    x[i] = i < n_turned ? z : x[i];
                }
                *reinterpret_cast<uint4*>(dst(h) + at) = a[k];
            }
        }
    } else {
        // A granule of eight features to a thread. Other threads of the warp may read what this one writes (in place), so a warp writes once all
        // its lanes have read; every lane stays for that.
        const int at = lane * 8;
        const bool in = token_in && at < p.head_dim;
        const int n_turned = max(0, min(8, p.rot - at));   // the others are passed on
        // The partners of features at .. at + 7 are at + pairs .. (first half) or at - pairs .. (second half); a granule that
        // holds features of both halves has partners of both kinds, eight of each
        const int up = at + pairs, down = at - pairs;
        const bool need_up = in && at < pairs && n_turned > 0;
        const bool need_down = in && at + n_turned > pairs && n_turned > 0;
        auto eight_from = [&](const half* x, int d) {   // features d .. d + 7 of a head, those outside of it as zeros
            const int g = d >> 3, shift = d & 7;        // (arithmetic: down to -1)
            const int last = (p.head_dim >> 3) - 1;
            uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
            if (g >= 0 && g <= last) lo = *reinterpret_cast<const uint4*>(x + g * 8);
            if (shift && g + 1 >= 0 && g + 1 <= last) hi = *reinterpret_cast<const uint4*>(x + g * 8 + 8);
            uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            if (shift & 4)
#pragma unroll
                for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
            if (shift & 2)
#pragma unroll
                for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
            uint4 r;
            r.x = (shift & 1) ? __funnelshift_r(w[0], w[1], 16) : w[0];
            r.y = (shift & 1) ? __funnelshift_r(w[1], w[2], 16) : w[1];
            r.z = (shift & 1) ? __funnelshift_r(w[2], w[3], 16) : w[2];
            r.w = (shift & 1) ? __funnelshift_r(w[3], w[4], 16) : w[3];
            return r;
        };
        uint4 a[kHeadsInFlight], bu[kHeadsInFlight], bd[kHeadsInFlight];
        auto fetch = [&](int h0) {
#pragma unroll
            for (int k = 0; k < kHeadsInFlight; ++k) {
                const int h = h0 + k * head_step;
                if (!in || h >= heads) continue;
                a[k] = *reinterpret_cast<const uint4*>(src(h) + at);
                bu[k] = bd[k] = make_uint4(0u, 0u, 0u, 0u);
                if (need_up) bu[k] = eight_from(src(h), up);
                if (need_down) bd[k] = eight_from(src(h), down);
            }
        };
        fetch(first_head);
        take_angles();
        float c[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = at + i;
            const bool second = d >= pairs;
            const int pair = second ? d - pairs : d;
            const float2 v = cs[i < n_turned ? pair : 0];
            c[i] = v.x;
            s[i] = second ? v.y : -v.y;
        }
        const int iterations = (heads + head_step * kHeadsInFlight - 1) / (head_step * kHeadsInFlight);
        for (int n = 0; n < iterations; ++n) {
            const int h0 = first_head + n * head_step * kHeadsInFlight;
            if (n) fetch(h0);
            __syncwarp();
#pragma unroll
            for (int k = 0; k < kHeadsInFlight; ++k) {
                const int h = h0 + k * head_step;
                if (!in || h >= heads) continue;
                float x[8], partner[8], z[8];
                unpack8(a[k], x);
                float u[8], d[8];
                unpack8(bu[k], u);
                unpack8(bd[k], d);
#pragma unroll
                for (int i = 0; i < 8; ++i) partner[i] = at + i < pairs ? u[i] : d[i];
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = i < n_turned ? x[i] * c[i] + partner[i] * s[i] : x[i];
                *reinterpret_cast<uint4*>(dst(h) + at) = pack8(z);
            }
        }
    }
}

}  // namespace
}  // namespace et

extern "C" int et_rotary_axes(void* q_out, const void* q, int q_out_pitch, int q_pitch, int nhead_q, void* k_out, const void* k, int k_out_pitch,
                              int k_pitch, int nhead_k, int head_dim, int rot_dim, const int* positions, int n_axes, const float* inv_freq,
                              const int* axis, int interleaved, int tokens, void* stream) {
    using namespace et;
    ET_REQUIRE(tokens >= 0 && nhead_q >= 0 && nhead_k >= 0, "et_rotary_axes: negative size");
    ET_REQUIRE(head_dim >= 2 && head_dim <= 256, "et_rotary_axes: head_dim must be 2 to 256");
    ET_REQUIRE(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 2 == 0, "et_rotary_axes: rot_dim must be even and at most head_dim");
    ET_REQUIRE(n_axes >= 1, "et_rotary_axes: at least one axis");
    ET_REQUIRE((long long)nhead_q * head_dim <= 0x7fffffff && (long long)nhead_k * head_dim <= 0x7fffffff, "et_rotary_axes: too many heads");
    if (tokens == 0 || nhead_q + (long long)nhead_k == 0) return ET_OK;
    ET_REQUIRE((nhead_q == 0 || (q && q_out)) && (nhead_k == 0 || (k && k_out)), "et_rotary_axes: null pointer");
    ET_REQUIRE(rot_dim == 0 || (positions && inv_freq && axis), "et_rotary_axes: null pointer");
    ET_REQUIRE(nhead_q == 0 || (q_pitch >= nhead_q * head_dim && q_out_pitch >= nhead_q * head_dim), "et_rotary_axes: pitch below the width of the heads");
    ET_REQUIRE(nhead_k == 0 || (k_pitch >= nhead_k * head_dim && k_out_pitch >= nhead_k * head_dim), "et_rotary_axes: pitch below the width of the heads");
    // a result may lie where its input lies, row for row; any other overlap would be read after it is written
    ET_REQUIRE(nhead_q == 0 || q != q_out || q_pitch == q_out_pitch, "et_rotary_axes: in place the pitches must be equal");
    ET_REQUIRE(nhead_k == 0 || k != k_out || k_pitch == k_out_pitch, "et_rotary_axes: in place the pitches must be equal");
    ET_REQUIRE(nhead_q + (long long)nhead_k <= 0xffff, "et_rotary_axes: too many heads");
    RotaryParams p;
    p.q_out = static_cast<half*>(q_out); p.k_out = static_cast<half*>(k_out);
    p.q = static_cast<const half*>(q); p.k = static_cast<const half*>(k);
    p.q_out_pitch = q_out_pitch; p.q_pitch = q_pitch; p.k_out_pitch = k_out_pitch; p.k_pitch = k_pitch;
    p.positions = positions; p.inv_freq = inv_freq; p.axis = axis;
    p.nhead_q = nhead_q; p.nhead_k = nhead_k; p.head_dim = head_dim; p.rot = rot_dim; p.n_axes = n_axes; p.tokens = tokens;
    p.interleaved = interleaved != 0;
    p.in_place_q = q == q_out; p.in_place_k = k == k_out;
    auto granules = [](const void* a, const void* b, int pa, int pb) { return aligned16(a) && aligned16(b) && pa % 8 == 0 && pb % 8 == 0; };
    const bool vec = head_dim % 8 == 0 && (nhead_q == 0 || granules(q, q_out, q_pitch, q_out_pitch)) && (nhead_k == 0 || granules(k, k_out, k_pitch, k_out_pitch));
    const int pairs = rot_dim / 2;
    const int pairing = !vec ? kScalar : p.interleaved ? kNeighbours : pairs % 8 == 0 ? kHalves8 : kHalves;
    const int want = pairing == kScalar ? min(32, max(1, pairs)) : pairing == kHalves8 ? pairs / 8 + (head_dim - rot_dim) / 8 : head_dim / 8;
    p.lanes = 1;
    while (p.lanes < want) p.lanes *= 2;
    if (pairing == kHalves8 || pairing == kNeighbours) p.lanes = want;   // (5003 tokens of 40 heads of 128, 96 features turned: ten lanes 21.4 us, sixteen 32)
    // A thread has kHeadsInFlight heads, all requested at once, one where there are few tokens; a block has as many tokens as make 128 threads, but no more
    // than leave every SM eight blocks. (32768 tokens of 32 heads of 64 in blocks of 128, 256, 512 threads: 42.7, 45.0, 61.1 us, with two heads to a thread 44.4,
    // three 45.4, four 41.9, neighbours with four, six, eight 41.0, 43.0, 42.3; 4000 tokens of 24 heads with four blocks to an SM 7.2, eight 6.8; 64 tokens
    // of 24 heads with one, two, four, eight heads: 2.2, 2.2, 2.9, 4.2.)
    const int heads = nhead_q + nhead_k, in_flight = tokens > sm_count() * 4 ? kHeadsInFlight : 1;
    p.head_step = max(1, min((heads + in_flight - 1) / in_flight, kMaxThreads / p.lanes));
    p.block_tokens = max(1, min(128 / (p.head_step * p.lanes), tokens / (sm_count() * 8)));
    const int threads = (p.block_tokens * p.head_step * p.lanes + 31) / 32 * 32;
    const int blocks = (tokens + p.block_tokens - 1) / p.block_tokens;
    const size_t smem = (size_t)p.block_tokens * max(pairs, 1) * sizeof(float2);
    const auto kernel = pairing == kScalar ? rotary_kernel<kScalar> : pairing == kHalves8 ? rotary_kernel<kHalves8> : pairing == kHalves ? rotary_kernel<kHalves> : rotary_kernel<kNeighbours>;
    return cuda_status(launch_pdl(kernel, dim3(blocks), dim3(threads), smem, static_cast<cudaStream_t>(stream), p), "et_rotary_axes launch");
}

extern "C" int et_rotary_axes_by(const et_rotary_axes_args* a) {
    ET_REQUIRE(a, "et_rotary_axes_by: null pointer");
    return et_rotary_axes(a->q_out, a->q, a->q_out_pitch, a->q_pitch, a->nhead_q, a->k_out, a->k, a->k_out_pitch, a->k_pitch, a->nhead_k, a->head_dim, a->rot_dim, a->positions,
                          a->n_axes, a->inv_freq, a->axis, a->interleaved, a->tokens, a->stream);
}
