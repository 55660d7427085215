// Device-side append of a ragged batch of new tokens (prompts and single tokens) to the latent
// cache, with the latent's RMS norm and the rotary position rotation of the key and the queries
// applied on the way. Token t = cu[b] + i of sequence b has position p = lens[b] + i:
//   cache[row(b, p)][0 : dc]       = c[t] * rsqrt(mean(c[t]^2) + eps) * w   (w given; else c[t])
//   cache[row(b, p)][dc : dc + dR] = rot(k[t], p)
//   q_out[t][h]                    = rot(q[t][h], p)
//   rot(x, p)[i] = x[i] cos - x[i + dR/2] sin,  rot(x, p)[i + dR/2] = x[i] sin + x[i + dR/2] cos
// The sums and products are in fp32; each result is rounded once, to the cache's 16-bit type.
//
// Bound by the bytes (about 2 (dc + dR + H dR) 2 bytes a token, a few flop each), and by latency for
// a handful of tokens. One warp does one piece of one token: its cache row, or up to 32 heads of its
// queries, so that a single token with many heads also spreads over the GPU; nothing is shared
// between warps, and every value is read and written once, as 16-byte vectors. A warp issues its
// data loads before it looks its sequence up, so the look-up's latency is not added to theirs.
#include <cmath>

#include "mla_internal.cuh"
#include "ops.cuh"

namespace mla {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kHeadsPerTask = 32;
constexpr int kRowVecs = 4;   // 16-byte vectors of a latent per lane: dc <= 32 * 8 * 4 = 1024

// Index of the sequence whose tokens [cu[b], cu[b + 1]) hold t, or -1. Warp-wide search: 32 probes a
// round (cu is non-decreasing; whatever it holds, the probes stay in [0, B)).
__device__ __forceinline__ int find_seq(const int* __restrict__ cu, int B, int t, int lane) {
    int lo = 0, n = B;
    do {
        const int step = (n + 31) / 32;
        const bool le = lane * step < n && cu[lo + lane * step] <= t;
        const int k = __popc(__ballot_sync(0xffffffffu, le));
        if (k == 0) return -1;
        lo += (k - 1) * step;
        n = min(step, n - (k - 1) * step);
    } while (n > 1);
    return cu[lo] <= t && t < cu[lo + 1] ? lo : -1;
}

// Position and cache row of token t: pos < 0 when the token has no place (no sequence, a full or
// broken one), row < 0 when its page or offset lies outside the cache.
__device__ __forceinline__ void place(const AppendRope& A, int t, int lane, int* pos, long long* row) {
    *pos = -1;
    *row = -1;
    const int b = find_seq(A.cu, A.B, t, lane);
    if (b < 0) return;
    const int len = A.lens[b];
    const long long p = static_cast<long long>(len) + (t - A.cu[b]);
    if (len < 0 || p >= A.max_len) return;
    *pos = static_cast<int>(p);
    long long r;
    if (A.pages) {
        const int pg = A.pages[static_cast<long long>(b) * A.max_pages + *pos / A.page_rows];
        r = static_cast<long long>(pg) * A.page_rows + *pos % A.page_rows;
        if (pg < 0) r = -1;
    } else {
        r = (A.offs ? A.offs[b] : static_cast<long long>(b) * A.max_len) + p;
    }
    *row = r >= 0 && r < A.kv_rows ? r : -1;
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = ElemTraits<T>::to_f2(*reinterpret_cast<const typename ElemTraits<T>::T2*>(&x[i]));
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    alignas(16) T y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = ElemTraits<T>::from_f(f[i]);
    return *reinterpret_cast<const uint4*>(y);
}

// cos and sin of rope pairs i0 .. i0 + 7 at position pos
__device__ __forceinline__ void angles8(const AppendRope& A, int pos, int i0, float (&c)[8], float (&s)[8]) {
    if (A.cos) {
        const long long at = static_cast<long long>(pos) * (A.dR / 2) + i0;
        const float4* c4 = reinterpret_cast<const float4*>(A.cos + at);
        const float4* s4 = reinterpret_cast<const float4*>(A.sin + at);
        const float4 c0 = __ldg(c4), c1 = __ldg(c4 + 1), s0 = __ldg(s4), s1 = __ldg(s4 + 1);
        c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
        s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) rope_sincos_exact(pos, A.freq[i0 + i], &s[i], &c[i]);
    }
}

template <typename T>
__device__ __forceinline__ void rotate8(uint4& lo, uint4& hi, const float (&c)[8], const float (&s)[8]) {
    float a[8], b[8], x[8], y[8];
    unpack8<T>(lo, a);
    unpack8<T>(hi, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = a[i] * c[i] - b[i] * s[i];
        y[i] = a[i] * s[i] + b[i] * c[i];
    }
    lo = pack8<T>(x);
    hi = pack8<T>(y);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// 16-byte path: dc % 8 == 0, dc <= 1024, dR % 16 == 0, every pointer and stride a multiple of 16 bytes.
template <typename T>
__device__ __forceinline__ void append_task_vec(const AppendRope& A, int t, int part, int lane) {
    const int nu = A.dR / 16;   // (lo, hi) vector pairs of a rotated row
    int pos;
    long long row;
    if (part == 0) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(A.c) + t * A.c_stride);
        const uint4* ksrc = reinterpret_cast<const uint4*>(static_cast<const T*>(A.k) + t * A.k_stride);
        const int nv = A.dc / 8;
        uint4 v[kRowVecs], lo, hi;
#pragma unroll
        for (int j = 0; j < kRowVecs; ++j)
            if (lane + 32 * j < nv) v[j] = src[lane + 32 * j];
        if (lane < nu) {
            lo = ksrc[lane];
            hi = ksrc[nu + lane];
        }
        place(A, t, lane, &pos, &row);
        if (row < 0) {
            if (lane == 0 && A.status) atomicOr(A.status, pos < 0 ? 1 : 2);
            return;
        }
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(A.kv) + row * A.stride);
        if (A.w) {
            const uint4* w4 = reinterpret_cast<const uint4*>(A.w);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < kRowVecs; ++j)
                if (lane + 32 * j < nv) {
                    float f[8];
                    unpack8<T>(v[j], f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum += f[i] * f[i];
                }
            const float r = rsqrtf(warp_sum(sum) / static_cast<float>(A.dc) + A.eps);
#pragma unroll
            for (int j = 0; j < kRowVecs; ++j)
                if (lane + 32 * j < nv) {
                    float f[8], w[8];
                    unpack8<T>(v[j], f);
                    unpack8<T>(__ldg(w4 + lane + 32 * j), w);
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = f[i] * r * w[i];
                    v[j] = pack8<T>(f);
                }
        }
#pragma unroll
        for (int j = 0; j < kRowVecs; ++j)
            if (lane + 32 * j < nv) dst[lane + 32 * j] = v[j];
        if (lane < nu) {
            float c[8], s[8];
            angles8(A, pos, 8 * lane, c, s);
            rotate8<T>(lo, hi, c, s);
            dst[nv + lane] = lo;
            dst[nv + nu + lane] = hi;
        }
        return;
    }
    // queries: lane = (head within a step, vector pair); a lane keeps its pair, so its angles serve
    // every head it takes
    const int hps = 32 / nu, u = lane % nu, hl = lane / nu;
    const int h1 = min(A.H, part * kHeadsPerTask);
    const T* q = static_cast<const T*>(A.q) + t * A.q_ts;
    T* qo = static_cast<T*>(A.qo) + t * A.qo_ts;
    constexpr int kSteps = 2;
    int h = (part - 1) * kHeadsPerTask + hl;
    bool first = true;
    float c[8], s[8];
    for (; h - hl < h1; h += kSteps * hps) {
        uint4 lo[kSteps], hi[kSteps];
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
            if (hl < hps && h + j * hps < h1) {
                const uint4* p = reinterpret_cast<const uint4*>(q + (h + j * hps) * A.q_hs);
                lo[j] = p[u];
                hi[j] = p[nu + u];
            }
        if (first) {
            place(A, t, lane, &pos, &row);
            if (pos < 0) return;   // reported by the token's row
            angles8(A, pos, 8 * u, c, s);
            first = false;
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
            if (hl < hps && h + j * hps < h1) {
                rotate8<T>(lo[j], hi[j], c, s);
                uint4* p = reinterpret_cast<uint4*>(qo + (h + j * hps) * A.qo_hs);
                p[u] = lo[j];
                p[nu + u] = hi[j];
            }
    }
}

// Any dimensions and alignment, element by element (12 prompts of up to 4099 tokens: 137 us, 33 as vectors).
template <typename T>
__device__ void append_task_any(const AppendRope& A, int t, int part, int lane) {
    int pos;
    long long row;
    place(A, t, lane, &pos, &row);
    const int half = A.dR / 2;
    auto rotate = [&](const T* x, T* y, int i) {
        float c, s;
        if (A.cos) {
            c = A.cos[static_cast<long long>(pos) * half + i];
            s = A.sin[static_cast<long long>(pos) * half + i];
        } else {
            rope_sincos_exact(pos, A.freq[i], &s, &c);
        }
        const float a = ElemTraits<T>::to_f(x[i]), b = ElemTraits<T>::to_f(x[half + i]);
        y[i] = ElemTraits<T>::from_f(a * c - b * s);
        y[half + i] = ElemTraits<T>::from_f(a * s + b * c);
    };
    if (part == 0) {
        if (row < 0) {
            if (lane == 0 && A.status) atomicOr(A.status, pos < 0 ? 1 : 2);
            return;
        }
        const T* src = static_cast<const T*>(A.c) + t * A.c_stride;
        T* dst = static_cast<T*>(A.kv) + row * A.stride;
        const T* w = static_cast<const T*>(A.w);
        float r = 1.f;
        if (w) {
            float sum = 0.f;
            for (int i = lane; i < A.dc; i += 32) {
                const float f = ElemTraits<T>::to_f(src[i]);
                sum += f * f;
            }
            r = rsqrtf(warp_sum(sum) / static_cast<float>(A.dc) + A.eps);
        }
        for (int i = lane; i < A.dc; i += 32)
            dst[i] = w ? ElemTraits<T>::from_f(ElemTraits<T>::to_f(src[i]) * r * ElemTraits<T>::to_f(w[i])) : src[i];
        const T* k = static_cast<const T*>(A.k) + t * A.k_stride;
        for (int i = lane; i < half; i += 32) rotate(k, dst + A.dc, i);
        return;
    }
    if (pos < 0) return;
    const int h1 = min(A.H, part * kHeadsPerTask);
    for (int h = (part - 1) * kHeadsPerTask; h < h1; ++h)
        for (int i = lane; i < half; i += 32)
            rotate(static_cast<const T*>(A.q) + t * A.q_ts + h * A.q_hs, static_cast<T*>(A.qo) + t * A.qo_ts + h * A.qo_hs, i);
}

// (four blocks an SM: prompts want warps in flight more than long ones; two blocks with four steps of
// heads at a time took 36.8 us for 12 prompts of up to 4099 tokens and 16 heads, four with two 32.4)
template <typename T, bool kVec>
__global__ void __launch_bounds__(kAppendThreads, 4) append_rope_kernel(const __grid_constant__ AppendRope A, int parts) {
    const long long warp = (static_cast<long long>(blockIdx.x) * kAppendThreads + threadIdx.x) / 32;
    const int lane = threadIdx.x & 31;
    if (A.new_lens) {
        for (long long b = static_cast<long long>(blockIdx.x) * kAppendThreads + threadIdx.x; b < A.B;
             b += static_cast<long long>(gridDim.x) * kAppendThreads) {
            const int len = A.lens[b];
            const int n = min(A.cu[b + 1], A.tokens) - min(A.cu[b], A.tokens);
            const long long to = static_cast<long long>(len) + max(n, 0);
            A.new_lens[b] = len < 0 || len >= A.max_len ? len : static_cast<int>(to < A.max_len ? to : A.max_len);
        }
    }
    if (warp >= static_cast<long long>(A.tokens) * parts) return;
    const int t = static_cast<int>(warp / parts), part = static_cast<int>(warp % parts);
    if constexpr (kVec) append_task_vec<T>(A, t, part, lane);
    else append_task_any<T>(A, t, part, lane);
}

template <typename T>
cudaError_t launch(const AppendRope& A, cudaStream_t s) {
    const int parts = 1 + (A.q ? ceil_div(A.H, kHeadsPerTask) : 0);
    const long long warps = static_cast<long long>(A.tokens) * parts;
    const long long blocks = (warps * 32 + kAppendThreads - 1) / kAppendThreads;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    auto a16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool vec = A.dc % 8 == 0 && A.dc <= 32 * 8 * kRowVecs && A.dR % 16 == 0 && A.stride % 8 == 0 &&
                     A.c_stride % 8 == 0 && A.k_stride % 8 == 0 && a16(A.kv) && a16(A.c) && a16(A.k) && a16(A.w) &&
                     a16(A.cos) && a16(A.sin) &&
                     (!A.q || (a16(A.q) && a16(A.qo) && A.q_ts % 8 == 0 && A.q_hs % 8 == 0 && A.qo_ts % 8 == 0 &&
                               A.qo_hs % 8 == 0));
    const dim3 grid(static_cast<unsigned>(blocks > 0 ? blocks : 1));
    if (vec) append_rope_kernel<T, true><<<grid, kAppendThreads, 0, s>>>(A, parts);
    else append_rope_kernel<T, false><<<grid, kAppendThreads, 0, s>>>(A, parts);
    count_launches(1);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append_rope(const AppendRope& A, bool bf16, cudaStream_t s) {
    return bf16 ? launch<__nv_bfloat16>(A, s) : launch<__half>(A, s);
}

}  // namespace mla
