// A shared projection with the requests' low-rank adapters beside it:
//     Y[m] = W x[m] + s_a B_a (A_a x[m]),   a = ids[m]   (no second term where a is no adapter)
// X (M, K), W (N, K), A (adapters, r, K), B (adapters, N, r), Y (M, N), all fp16 or bf16.
//
// Two kernels, the second launched beside the first (programmatic dependent launch):
//   1. lora_shrink_kernel: U = s_a A_a x[m] for each block of up to 256 tokens and each adapter that
//      occurs in it, one row per token and zeros for the other tokens, so that U is a matrix with the
//      active adapters' ranks as extra columns: the delta is U . [B_a1 | B_a2 | ..]^T, a product over
//      (active adapters x rank) more K columns of the same GEMM.
//   2. lora_gemm_kernel: Y^T tiles [128 weight rows x up to 256 tokens] on tcgen05, K columns first
//      (which need nothing of kernel 1), then the rank columns. Rank columns are taken 16 at a time
//      (one MMA K-step), so an adapter of rank 16 costs one step, and only the adapters that a block
//      of tokens really uses are read.
// Small batches are bound by W's bytes (each read once for all tokens), prompts by the tensor pipe.
//
// Work split: whole tiles go round robin over one CTA per SM; the tiles that do not fill a last
// round are cut along K into equal shares for all CTAs, so no SM idles. A CTA that shares a tile
// stores its fp32 partial and counts itself; the one that completes the count adds all partials in
// their order along K, so results do not depend on who came last. No CTA waits for another.
//
// A zero of U times an infinite or NaN value of another request's adapter would be NaN, so an output
// that is not finite is computed again from its own operands alone (own_element): a broken adapter
// stays with its requests, and only then costs more.
//
// Rounding: products and sums in fp32; U is rounded to the inputs' type once (it is an MMA operand)
// and Y once.
#include "mla_internal.cuh"
#include "ops.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

namespace mla {
using namespace sm100;

namespace {

constexpr int kRows = 128;            // weight rows per tile (MMA M)
constexpr int kMaxTok = 256;          // tokens per tile (MMA N)
constexpr int kChunk = 64;            // K elements per stage
constexpr int kStep = 16;             // K elements per MMA
constexpr int kGemmThreads = 192;     // warp 0 loads, warp 1 issues, warps 2-5 read out
constexpr int kSmemCap = 200 * 1024;
constexpr int kMinChunks = 4;         // shortest share of a cut tile
constexpr int kShrinkWarps = 16;
constexpr int kShrinkTok = 32;        // tokens per shrink block
enum : int { kWaitLoad = 1, kWaitMma = 3, kWaitAcc = 4, kWaitOut = 5 };

struct Plan {
    int M, N, K, r;
    int tb, nb;                       // tokens per block (a multiple of 16), blocks
    int adapters, slots, rsteps;      // most adapters of a block, MMA steps per adapter
    int kc, tiles;                    // K chunks, tiles (weight rows / 128 x blocks)
    int grid, full;                   // CTAs, whole tiles (a multiple of grid)
    int tail_ctas;                    // CTAs that share the other tiles
    int stages, stage_bytes;
    size_t off_status, off_count, off_meta, off_u, off_part, total;
};

int up(int a, int b) { return (a + b - 1) / b * b; }

Plan make_plan(int M, int N, int K, int adapters, int rank, int sms) {
    Plan p = {};
    p.M = M; p.N = N; p.K = K; p.r = rank; p.adapters = adapters;
    p.nb = ceil_div(M, kMaxTok);
    p.tb = up(ceil_div(M, p.nb), kStep);
    p.nb = ceil_div(M, p.tb);
    p.slots = adapters < p.tb ? adapters : p.tb;
    p.rsteps = ceil_div(rank, kStep);
    p.kc = ceil_div(K, kChunk);
    p.tiles = ceil_div(N, kRows) * p.nb;
    p.grid = sms;
    p.full = p.tiles / p.grid * p.grid;
    const int rest = p.tiles - p.full;
    const long long chunks = static_cast<long long>(rest) * p.kc;
    long long ctas = chunks / kMinChunks;
    if (ctas > p.grid) ctas = p.grid;
    if (ctas < rest) ctas = rest;
    p.tail_ctas = static_cast<int>(ctas);
    if (p.full == 0) p.grid = p.tail_ctas;
    p.stage_bytes = (kRows + p.tb) * 128;
    p.stages = kSmemCap / p.stage_bytes;
    if (p.stages > 10) p.stages = 10;
    auto a256 = [](size_t x) { return (x + 255) / 256 * 256; };
    size_t off = 0;
    p.off_status = off; off += 256;
    p.off_count = off; off = a256(off + sizeof(int) * static_cast<size_t>(p.grid));
    p.off_meta = off; off = a256(off + sizeof(int) * static_cast<size_t>(p.nb) * (p.slots + 1));
    p.off_u = off; off = a256(off + static_cast<size_t>(p.nb) * p.slots * p.rsteps * p.tb * kStep * 2);
    p.off_part = off;
    if (rest > 0 && p.tail_ctas > rest) off += static_cast<size_t>(p.tail_ctas) * 2 * kRows * p.tb * sizeof(float);
    p.total = a256(off);
    return p;
}

template <typename T> struct Fmt;
template <> struct Fmt<__half> { static constexpr uint32_t v = 0; };
template <> struct Fmt<__nv_bfloat16> { static constexpr uint32_t v = 1; };

// ------------------------------------------------------------------------------------- shrink

// D (16 x 8) += A (16 x 16) B (16 x 8)
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                        uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Block (unit, rank step, token block). A unit is one adapter of the token block with up to 32 of
// its tokens. 16 warps cut K; each holds the 16 ranks x 32 tokens in registers as warp-level MMA
// tiles and reads A's and x's rows straight from global memory, 16 bytes a lane: the sum over K may
// take its columns in any order, so lane t of a quad takes columns 8 t .. 8 t + 7 of each 32, for both
// operands alike. Tokens are gathered by their rows' addresses. The partial sums meet in shared
// memory in warp order. (16 ranks x 32 tokens are too small for tcgen05's 128-row tile, and the whole
// kernel is a few microseconds of latency beside the GEMM's start.)
template <typename T>
__global__ void __launch_bounds__(32 * kShrinkWarps) lora_shrink_kernel(const LoraArgs A, const Plan P, unsigned char* ws) {
    __shared__ __align__(16) int ids[kMaxTok];
    __shared__ int unit_id, unit_sub, unit_slot;
    __shared__ int warp_slots[8], warp_units[8];
    __shared__ int list[kShrinkTok];
    __shared__ float red[kShrinkWarps][kStep][kShrinkTok + 1];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int unit = blockIdx.x, q = blockIdx.y, blk = blockIdx.z;
    const int m0 = blk * P.tb, mt = min(P.tb, P.M - m0);
    if (tid < kMaxTok) {
        const int id = tid < mt ? A.ids[m0 + tid] : -1;
        ids[tid] = id >= 0 && id < P.adapters ? id : -1;
    }
    if (tid < kShrinkTok) list[tid] = -1;
    if (tid == 0) unit_id = -1;
    if (blockIdx.x + blockIdx.y + blockIdx.z == 0) {
        int* count = reinterpret_cast<int*>(ws + P.off_count);
        for (int i = tid; i < P.grid; i += blockDim.x) count[i] = 0;
        if (tid == 0) *reinterpret_cast<int*>(ws + P.off_status) = 0;
    }
    __syncthreads();
    // the block's adapters in order of their first token; a token's rank among its adapter's
    int id = -1, count = 0, rank_in = 0, first = kMaxTok;
    if (tid < kMaxTok && (id = ids[tid]) >= 0) {
        for (int j = 0; j < mt; ++j)
            if (ids[j] == id) {
                if (count == 0) first = j;
                rank_in += j < tid;
                ++count;
            }
    }
    const bool leader = id >= 0 && first == tid;
    const int groups = leader ? (count + kShrinkTok - 1) / kShrinkTok : 0;
    int s_incl = leader, u_incl = groups;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, s_incl, o), b = __shfl_up_sync(0xffffffffu, u_incl, o);
        if (lane >= o) {
            s_incl += a;
            u_incl += b;
        }
    }
    if (warp < 8 && lane == 31) {
        warp_slots[warp] = s_incl;
        warp_units[warp] = u_incl;
    }
    __syncthreads();
    if (warp < 8) {
        int s0 = 0, u0 = 0;
        for (int w = 0; w < warp; ++w) {
            s0 += warp_slots[w];
            u0 += warp_units[w];
        }
        const int slot = s0 + s_incl - 1, u1 = u0 + u_incl;
        if (leader && unit >= u1 - groups && unit < u1) {
            unit_id = id;
            unit_slot = slot;
            unit_sub = unit - (u1 - groups);
        }
        if (unit == 0 && q == 0) {
            int* meta = reinterpret_cast<int*>(ws + P.off_meta) + static_cast<size_t>(blk) * (P.slots + 1);
            if (leader) meta[1 + slot] = id;
            if (tid == kMaxTok - 1) meta[0] = slot + 1;
        }
    }
    __syncthreads();
    const int a = unit_id, sub = unit_sub;
    if (a < 0) return;
    if (tid < kMaxTok && id == a && rank_in / kShrinkTok == sub) list[rank_in % kShrinkTok] = tid;
    __syncthreads();
    T* u = reinterpret_cast<T*>(ws + P.off_u) +
           (static_cast<size_t>(blk) * P.slots * P.rsteps + unit_slot * P.rsteps + q) * P.tb * kStep;
    if (sub == 0)   // the other tokens' rows of this adapter's columns
        for (int i = tid; i < P.tb * 2; i += blockDim.x)
            if (ids[i / 2] != a) reinterpret_cast<uint4*>(u)[i] = make_uint4(0, 0, 0, 0);
    const int g = lane / 4, t = lane % 4;
    const T* arow[2];
    const T* xrow[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int k = q * kStep + g + 8 * i;
        arow[i] = k < P.r ? static_cast<const T*>(A.a) + (static_cast<long long>(a) * P.r + k) * P.K : nullptr;
    }
    int nt = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = list[8 * i + g];
        xrow[i] = m >= 0 ? static_cast<const T*>(A.x) + (m0 + m) * A.x_stride : nullptr;
        if (list[8 * i] >= 0) nt = i + 1;
    }
    float acc[4][4] = {};
    constexpr int kUnroll = 4;
    for (int k0 = 32 * warp; k0 < P.K; k0 += 32 * kShrinkWarps * kUnroll) {
        uint4 va[kUnroll][2], vx[kUnroll][4];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const int k = k0 + j * 32 * kShrinkWarps + 8 * t;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                va[j][i] = arow[i] && k < P.K ? __ldg(reinterpret_cast<const uint4*>(arow[i] + k)) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                vx[j][i] = xrow[i] && k < P.K ? __ldg(reinterpret_cast<const uint4*>(xrow[i] + k)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < nt) {
                    mma16816<T>(acc[i], va[j][0].x, va[j][1].x, va[j][0].y, va[j][1].y, vx[j][i].x, vx[j][i].y);
                    mma16816<T>(acc[i], va[j][0].z, va[j][1].z, va[j][0].w, va[j][1].w, vx[j][i].z, vx[j][i].w);
                }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        red[warp][g][8 * i + 2 * t] = acc[i][0];
        red[warp][g][8 * i + 2 * t + 1] = acc[i][1];
        red[warp][g + 8][8 * i + 2 * t] = acc[i][2];
        red[warp][g + 8][8 * i + 2 * t + 1] = acc[i][3];
    }
    __syncthreads();
    const int k = tid % kStep, m = list[tid / kStep];   // 512 threads: 16 ranks x 32 tokens
    if (m >= 0) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kShrinkWarps; ++w) v += red[w][k][tid / kStep];
        u[m * kStep + k] = ElemTraits<T>::from_f(A.scales ? v * A.scales[a] : v);
    }
}

// ------------------------------------------------------------------------------------- GEMM

struct Maps {
    CUtensorMap w, x, b, u;
};

// One piece of a CTA's work: chunks [c0, c1) of a tile's K columns.
struct Item {
    int tile, c0, c1;
    int j;           // index among the cut tiles, or -1
};
// Walks the CTA's pieces; every role walks an identical copy.
struct Walk {
    int next_full;
    long long c, c_end;
    __device__ explicit Walk(const Plan& P) {
        const int w = blockIdx.x;
        next_full = w;
        c = c_end = 0;
        if (w < P.tail_ctas) {
            const long long total = static_cast<long long>(P.tiles - P.full) * P.kc;
            c = total * w / P.tail_ctas;
            c_end = total * (w + 1) / P.tail_ctas;
        }
    }
    __device__ bool next(const Plan& P, Item* it) {
        if (next_full < P.full) {
            *it = {next_full, 0, P.kc, -1};
            next_full += P.grid;
            return true;
        }
        if (c >= c_end) return false;
        const int j = static_cast<int>(c / P.kc);
        const int c0 = static_cast<int>(c % P.kc);
        const int n = static_cast<int>(c_end - c);
        const int c1 = min(P.kc, c0 + n);
        *it = {P.full + j, c0, c1, j};
        c += c1 - c0;
        return true;
    }
};

struct __align__(8) Bars {
    uint64_t full[10], empty[10], acc_full[2], acc_empty[2];
    uint32_t tmem;
    int last;
};

__device__ __forceinline__ int code(int site) { return kStatusTimeout | (site << 8); }

// Output element (token m of the block, weight row n) from the token's own operands: the rare path of
// outputs that came out infinite or NaN.
template <typename T>
__device__ __noinline__ float own_element(const LoraArgs& A, const Plan& P, const unsigned char* ws, int blk, int m, int n) {
    const T* x = static_cast<const T*>(A.x) + static_cast<long long>(blk * P.tb + m) * A.x_stride;
    const T* w = static_cast<const T*>(A.w) + static_cast<long long>(n) * P.K;
    float v = 0.f;
    for (int k = 0; k < P.K; ++k) v = fmaf(ElemTraits<T>::to_f(x[k]), ElemTraits<T>::to_f(w[k]), v);
    const int id = A.ids[blk * P.tb + m];
    if (id < 0 || id >= P.adapters) return v;
    const int* meta = reinterpret_cast<const int*>(ws + P.off_meta) + static_cast<size_t>(blk) * (P.slots + 1);
    int slot = 0;
    while (slot < meta[0] && meta[1 + slot] != id) ++slot;
    const T* u = reinterpret_cast<const T*>(ws + P.off_u);
    const T* b = static_cast<const T*>(A.b) + (static_cast<long long>(id) * P.N + n) * P.r;
    for (int k = 0; k < P.r; ++k) {
        const size_t step = static_cast<size_t>(blk) * P.slots * P.rsteps + slot * P.rsteps + k / kStep;
        v = fmaf(ElemTraits<T>::to_f(u[(step * P.tb + m) * kStep + k % kStep]), ElemTraits<T>::to_f(b[k]), v);
    }
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kGemmThreads, 1)
lora_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Plan P,
                 const __grid_constant__ LoraArgs A, unsigned char* ws) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Bars* bars = reinterpret_cast<Bars*>(smem + P.stages * P.stage_bytes);
    const uint32_t ring = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* err = reinterpret_cast<int*>(ws + P.off_status);
    if (threadIdx.x == 0) {
        for (int s = 0; s < P.stages; ++s) {
            mbar_init(smem_u32(&bars->full[s]), 1);
            mbar_init(smem_u32(&bars->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&bars->acc_full[b]), 1);
            mbar_init(smem_u32(&bars->acc_empty[b]), 128);
        }
        fence_mbar_init();
        tma_prefetch_desc(&maps.w);
        tma_prefetch_desc(&maps.x);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&bars->tmem), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = bars->tmem;
    const int* meta = reinterpret_cast<const int*>(ws + P.off_meta);

    if (warp == 0) {
        // ---- loads
        if (lane == 0) {
            Walk walk(P);
            Item it;
            int i = 0;
            bool ok = true, waited = false;
            auto stage = [&](uint32_t* dst, uint32_t* fb) -> bool {
                const int s = i % P.stages;
                if (i >= P.stages && !mbar_wait(smem_u32(&bars->empty[s]), ((i / P.stages) - 1) & 1, err, code(kWaitLoad)))
                    return false;
                *fb = smem_u32(&bars->full[s]);
                *dst = ring + s * P.stage_bytes;
                ++i;
                return true;
            };
            while (ok && walk.next(P, &it)) {
                const int n0 = it.tile / P.nb * kRows, blk = it.tile % P.nb;
                uint32_t dst, fb;
                for (int c = it.c0; c < it.c1; ++c) {
                    if (!(ok = stage(&dst, &fb))) break;
                    mbar_arrive_expect_tx(fb, static_cast<uint32_t>(P.stage_bytes));
                    tma_load_2d(dst, &maps.w, fb, kChunk * c, n0);
                    tma_load_2d(dst + kRows * 128, &maps.x, fb, kChunk * c, blk * P.tb);
                }
                if (!ok || it.c1 < P.kc) continue;
                if (!waited) {
                    pdl_wait();   // U and the adapters' list come from the shrink kernel
                    waited = true;
                }
                const int* m = meta + static_cast<size_t>(blk) * (P.slots + 1);
                const int steps = m[0] * P.rsteps;
                for (int s0 = 0; s0 < steps; s0 += 4) {
                    if (!(ok = stage(&dst, &fb))) break;
                    const int n = min(4, steps - s0);
                    mbar_arrive_expect_tx(fb, static_cast<uint32_t>(n * (kRows + P.tb) * 32));
                    for (int k = 0; k < n; ++k) {
                        const int slot = (s0 + k) / P.rsteps, q = (s0 + k) % P.rsteps;
                        tma_load_3d(dst + k * kRows * 32, &maps.b, fb, q * kStep, n0, m[1 + slot]);
                        tma_load_2d(dst + kRows * 128 + k * P.tb * 32, &maps.u, fb, 0,
                                    (blk * P.slots * P.rsteps + s0 + k) * P.tb);
                    }
                }
            }
            if (!waited) pdl_wait();
            // no load may still be in flight when shared memory is released
            for (int k = i > P.stages ? i - P.stages : 0; k < i; ++k)
                mbar_wait(smem_u32(&bars->full[k % P.stages]), (k / P.stages) & 1, err, code(kWaitLoad), 100000000ull);
        }
    } else if (warp == 1) {
        // ---- MMAs
        if (lane == 0) {
            Walk walk(P);
            Item it;
            int i = 0, n = 0;
            bool ok = true, waited = false;
            for (; ok && walk.next(P, &it); ++n) {
                const int blk = it.tile % P.nb;
                const int toks = min(P.tb, P.M - blk * P.tb);
                const uint32_t idesc = idesc_f16(kRows, (toks + 15) / 16 * 16, Fmt<T>::v, false, false);
                const uint32_t d = tbase + 256 * (n & 1);
                if (n >= 2 && !(ok = mbar_wait(smem_u32(&bars->acc_empty[n & 1]), ((n >> 1) - 1) & 1, err, code(kWaitAcc)))) break;
                tc_fence_after();
                uint32_t acc = 0;
                for (int c = it.c0; c < it.c1; ++c, ++i) {
                    const int s = i % P.stages;
                    if (!(ok = mbar_wait(smem_u32(&bars->full[s]), (i / P.stages) & 1, err, code(kWaitMma)))) break;
                    tc_fence_after();
                    const uint32_t a = ring + s * P.stage_bytes;
                    const uint64_t ad = smem_desc_sw128(a, 16, 1024), bd = smem_desc_sw128(a + kRows * 128, 16, 1024);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mma_ss(d, ad + static_cast<uint64_t>(2 * k), bd + static_cast<uint64_t>(2 * k), idesc, acc);
                        acc = 1;
                    }
                    mma_commit(smem_u32(&bars->empty[s]));
                }
                if (ok && it.c1 == P.kc) {
                    if (!waited) {
                        pdl_wait();
                        waited = true;
                    }
                    const int steps = meta[static_cast<size_t>(blk) * (P.slots + 1)] * P.rsteps;
                    for (int s0 = 0; s0 < steps; s0 += 4, ++i) {
                        const int s = i % P.stages;
                        if (!(ok = mbar_wait(smem_u32(&bars->full[s]), (i / P.stages) & 1, err, code(kWaitMma)))) break;
                        tc_fence_after();
                        const uint32_t a = ring + s * P.stage_bytes;
                        for (int k = 0; k < min(4, steps - s0); ++k)
                            mma_ss(d, smem_desc_sw32(a + k * kRows * 32), smem_desc_sw32(a + kRows * 128 + k * P.tb * 32),
                                   idesc, 1u);
                        mma_commit(smem_u32(&bars->empty[s]));
                    }
                }
                mma_commit(smem_u32(&bars->acc_full[n & 1]));
            }
        }
    } else {
        // ---- read-out: thread = weight row = TMEM lane
        const int row = (warp & 3) * 32 + lane;
        const uint32_t trow = tbase + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
        Walk walk(P);
        Item it;
        bool ok = true;
        pdl_wait();   // the partials' counters are cleared by the shrink kernel
        for (int n = 0; walk.next(P, &it); ++n) {
            const int blk = it.tile % P.nb, m0 = blk * P.tb, toks = min(P.tb, P.M - m0);
            const int col = it.tile / P.nb * kRows + row;
            const uint32_t d = trow + 256 * (n & 1);
            const bool got = mbar_wait(smem_u32(&bars->acc_full[n & 1]), (n >> 1) & 1, err, code(kWaitOut));
            ok = __all_sync(0xffffffffu, got) && ok;
            tc_fence_after();
            T* out = static_cast<T*>(A.y) + static_cast<long long>(m0) * P.N + col;
            auto store = [&](int m, float v) {
                if (!isfinite(v) && ok && meta[static_cast<size_t>(blk) * (P.slots + 1)] > 0)
                    v = own_element<T>(A, P, ws, blk, m, col);
                out[static_cast<long long>(m) * P.N] = ElemTraits<T>::from_f(v);
            };
            // the CTAs that share the tile
            int w0 = blockIdx.x, w1 = blockIdx.x;
            const long long total = static_cast<long long>(P.tiles - P.full) * P.kc;
            if (it.j >= 0) {
                w0 = static_cast<int>(((static_cast<long long>(it.j) * P.kc + 1) * P.tail_ctas - 1) / total);
                w1 = static_cast<int>(((static_cast<long long>(it.j) + 1) * P.kc * P.tail_ctas - 1) / total);
            }
            if (w0 == w1) {
                for (int m = 0; m < toks; m += 16) {
                    uint32_t v[16];
                    tmem_ld16_sync(d + m, v);
                    if (col < P.N)
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (m + k < toks) store(m + k, ok ? __uint_as_float(v[k]) : NAN);
                }
                tc_fence_before();
                mbar_arrive(smem_u32(&bars->acc_empty[n & 1]));
                continue;
            }
            float* parts = reinterpret_cast<float*>(ws + P.off_part);
            auto part = [&](int w) -> float* {
                // a CTA touches at most two cut tiles: the first into its slot 0, the second into slot 1
                const int first = static_cast<int>(total * w / P.tail_ctas / P.kc);
                return parts + (static_cast<size_t>(w) * 2 + (first == it.j ? 0 : 1)) * kRows * P.tb;
            };
            float* mine = part(blockIdx.x);
            for (int m = 0; m < toks; m += 16) {
                uint32_t v[16];
                tmem_ld16_sync(d + m, v);
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    mine[(m + k) * kRows + row] = ok ? __uint_as_float(v[k]) : NAN;
            }
            tc_fence_before();
            mbar_arrive(smem_u32(&bars->acc_empty[n & 1]));
            __threadfence();
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (threadIdx.x == 64) {
                int* count = reinterpret_cast<int*>(ws + P.off_count) + it.j;
                bars->last = atomicAdd(count, 1) == w1 - w0;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (!bars->last) continue;
            __threadfence();
            for (int m = 0; m < toks; m += 8) {
                float v[8] = {};
                for (int w = w0; w <= w1; ++w) {
                    const float* src = part(w) + m * kRows + row;
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] += __ldcg(src + k * kRows);   // tb is a multiple of 16
                }
                if (col < P.N)
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (m + k < toks) store(m + k, v[k]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tbase, 512);
    }
}

template <typename T>
cudaError_t launch(const LoraArgs& A, unsigned char* ws, int sms, cudaStream_t s) {
    const Plan P = make_plan(A.M, A.N, A.K, A.adapters, A.rank, sms);
    Maps maps;
    const uint64_t K = static_cast<uint64_t>(A.K), N = static_cast<uint64_t>(A.N), r = static_cast<uint64_t>(A.rank);
    const uint64_t wd[2] = {K, N}, ws1[1] = {K * 2};
    const uint64_t xd[2] = {K, static_cast<uint64_t>(A.M)}, xs[1] = {static_cast<uint64_t>(A.x_stride) * 2};
    const uint64_t bd[3] = {r, N, static_cast<uint64_t>(A.adapters)}, bs[2] = {r * 2, r * N * 2};
    const uint64_t ud[2] = {kStep, static_cast<uint64_t>(P.nb) * P.slots * P.rsteps * P.tb}, us[1] = {kStep * 2};
    const uint32_t tb = static_cast<uint32_t>(P.tb);
    const uint32_t wb[2] = {kChunk, kRows}, xb[2] = {kChunk, tb}, bb[3] = {kStep, kRows, 1}, ub[2] = {kStep, tb};
    if (!encode_tmap_16b(&maps.w, A.w, 2, wd, ws1, wb, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tmap_16b(&maps.x, A.x, 2, xd, xs, xb, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tmap_16b(&maps.b, A.b, 3, bd, bs, bb, CU_TENSOR_MAP_SWIZZLE_32B) ||
        !encode_tmap_16b(&maps.u, ws + P.off_u, 2, ud, us, ub, CU_TENSOR_MAP_SWIZZLE_32B))
        return cudaErrorInvalidValue;
    const int units = P.slots + P.tb / kShrinkTok;
    lora_shrink_kernel<T><<<dim3(units, P.rsteps, P.nb), 32 * kShrinkWarps, 0, s>>>(A, P, ws);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int smem = P.stages * P.stage_bytes + static_cast<int>(sizeof(Bars)) + 1024;
    e = ensure_dynamic_smem(reinterpret_cast<const void*>(lora_gemm_kernel<T>), kSmemCap + static_cast<int>(sizeof(Bars)) + 1024);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(P.grid);
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, lora_gemm_kernel<T>, maps, P, A, ws);
    count_launches(2);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

size_t lora_workspace(int M, int N, int K, int adapters, int rank, int sms) {
    return make_plan(M, N, K, adapters, rank, sms).total;
}

cudaError_t launch_lora(const LoraArgs& A, bool bf16, void* workspace, int sms, cudaStream_t s) {
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    return bf16 ? launch<__nv_bfloat16>(A, ws, sms, s) : launch<__half>(A, ws, sms, s);
}

}  // namespace mla
