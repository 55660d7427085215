// A shared projection with the requests' low-rank adapters beside it:
//     Y[m] = W x[m] + s_a B_a (A_a x[m]),   a = ids[m]   (no second term where a is no adapter)
// X (M, K), W (N, K), A (adapters, r, K), B (adapters, N, r), Y (M, N), all fp16 or bf16.
//
// Two kernels, the second let in while the first still runs (programmatic dependent launch):
//   1. lora_shrink_kernel: U = s_a A_a x[m], for each block of up to 256 tokens and each adapter that
//      occurs in it. A single block of more than 128 tokens is also put in adapter order (the rows of X
//      are copied): its MMAs then cover few columns that are not the adapter's.
//   2. lora_gemm_kernel: Y^T tiles [256 weight rows x up to 256 tokens] on tcgen05, a pair of CTAs each
//      (cta_group::2: 128 weight rows and half of the tokens' rows in each CTA's shared memory, so that
//      a token's row is loaded once for 256 weight rows). First the K columns, then the ranks as extra
//      K columns: for each active adapter a product of B_a's 256 rows with U's rows of the adapter's
//      tokens, added into those tokens' columns only. Only the adapters that a block really uses are
//      read, and an MMA covers whole groups of 32 columns.
//      Or lora_gemv_kernel on the CUDA cores, for one or two tokens.
// Small batches are bound by W's bytes (each read once for all tokens), prompts by the tensor pipe and
// by what L2 delivers to the SMs (without multicast a pair needs 62 KB for 0.5 us of MMAs). Without
// adapters the GEMM takes 212 us for 256 tokens onto 65536 rows of 7168 (1.14 PFLOP/s) and 266 us for
// 2051 tokens onto 5120 rows of 16384; with 32 adapters of rank 64 and 4 of rank 32 it is 267 and 298 us,
// of which 23 and 49 us are the shrink kernel's (replayed graphs; in a stream of calls, at the clocks that
// it settles at, 313 and 351).
//
// Work split: whole tiles go round robin over the pairs, and the tiles that do not fill a last round are
// cut. Blocks of 128 tokens and more are cut by columns (no sums to join: 256
// tokens onto 65536 rows 281 us, cut along K 298). Smaller ones, which W's bytes bound, are cut along K
// into equal shares for all pairs. A CTA that shares such a tile stores its fp32 partial and counts
// itself, per 32 columns; the one that completes a count adds all partials in their order along K, so
// results do not depend on who came last. No CTA waits for another pair's.
//
// A zero of U times an infinite or NaN value of another request's adapter would be NaN, so an output
// that is not finite is computed again from its own operands alone (own_columns): a broken adapter
// stays with its requests, and only then costs more.
//
// Rounding: products and sums in fp32; U is rounded to the inputs' type once where it is an MMA operand
// (fp16: in steps of 2^-24 below 2^-14; where it passes 65504, the outputs that use it are computed again
// from U in fp32, as the CUDA-core kernel does for its few tokens), and Y once.
#include "mla_internal.cuh"
#include "ops.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

#include <cstddef>

namespace mla {
using namespace sm100;

namespace {

constexpr int kRows = 128;            // weight rows per CTA (256 per pair and tile)
constexpr int kMaxTok = 256;          // tokens per tile (MMA N)
constexpr int kChunk = 64;            // K elements per 128-byte row
constexpr int kGroup = 2;             // chunks per stage
constexpr int kStep = 16;             // K elements per MMA
constexpr int kColStep = 32;          // an MMA of a CTA pair covers a multiple of 32 columns, from one on
constexpr int kGemmThreads = 192;     // warp 0 loads, warp 1 issues, warps 2-5 read out
constexpr int kSmemCap = 192 * 1024;  // leaves room for a block of the shrink kernel on the SM
constexpr int kMaxStages = 6;
constexpr int kMinChunks = 4;         // shortest share of a cut tile
constexpr int kSliceTok = 128;        // blocks of at least so many tokens are cut by columns
constexpr int kFewTokens = 2;         // up to so many tokens take the CUDA-core kernel (8192 x 5120, rank 16: one token
                                      // 16.8 us and 31 on the MMAs, two 22.6 and 29, four 38 and 29)
constexpr int kGemvWarps = 8, kGemvBlocks = 4;
constexpr int kGemvSteps = 2;         // 512-byte steps of a weight row in flight
constexpr int kSortTok = 128;         // a single block of more tokens is put in adapter order
constexpr int kMinSlice = 32;         // narrowest slice (648 tokens onto 804 rows of 15848: 64: 74 us, 32: 67)
constexpr int kJoinCols = 32;         // columns of a tile cut along K that are counted and added at a time
constexpr int kJoins = kSliceTok / kJoinCols;
constexpr int kShrinkWarps = 8;
constexpr int kShrinkTok = 32;        // tokens per shrink cluster
constexpr int kTable = 1024;          // adapters that the shrink kernel counts in a table
enum : int { kWaitLoad = 1, kWaitMma = 3, kWaitAcc = 4, kWaitOut = 5 };

struct Plan {
    int M, N, K, r;
    int tb, nb;                       // tokens per block (a multiple of 32), blocks
    int sorted;                       // one block, its columns in adapter order
    int adapters, slots, rsteps;      // most adapters of a block, MMA steps per adapter
    int kw, rchunks;                  // ranks per row of B's and U's tiles (16, 32 or 64), tiles per adapter
    int kc, tiles;                    // K chunks, tiles (weight rows / 256 x blocks)
    int pairs, full;                  // CTA pairs, whole tiles (a multiple of pairs)
    int slices, slice;                // column slices that the other tiles are cut into, 0: along K; their width
    int tail_pairs;                   // pairs that share the other tiles
    int width;                        // most columns of a piece
    int stages, stage_bytes;
    int ksplit, clusters, per_blk;    // CTAs of a shrink cluster, clusters in all and per token block
    size_t off_status, off_count, off_meta, off_perm, off_x, off_u, off_u32, off_part, total;
};

int up(int a, int b) { return (a + b - 1) / b * b; }

// Rank steps of a shrink item: x's rows are read once for all of them.
int shrink_steps(int rsteps) { return rsteps > 2 ? 4 : rsteps > 1 ? 2 : 1; }

Plan make_plan(int M, int N, int K, int adapters, int rank, int sms) {
    Plan p = {};
    p.M = M; p.N = N; p.K = K; p.r = rank; p.adapters = adapters;
    p.nb = ceil_div(M, kMaxTok);
    p.tb = up(ceil_div(M, p.nb), kColStep);
    p.nb = ceil_div(M, p.tb);
    // with up to 128 tokens an MMA over all columns costs less than the copy of X
    p.sorted = p.nb == 1 && p.tb > kSortTok;
    p.slots = adapters < p.tb ? adapters : p.tb;
    p.rsteps = ceil_div(rank, kStep);
    p.kw = rank > 32 ? 64 : rank > 16 ? 32 : 16;
    p.rchunks = ceil_div(rank, p.kw);
    p.kc = ceil_div(K, kChunk);
    p.tiles = ceil_div(N, 2 * kRows) * p.nb;
    p.pairs = sms / 2;
    p.full = p.tiles / p.pairs * p.pairs;
    const int rest = p.tiles - p.full;
    if (p.tb >= kSliceTok) {
        p.slices = rest == 0 ? 1 : p.pairs / rest < p.tb / kMinSlice ? p.pairs / rest : p.tb / kMinSlice;
        p.slice = up(ceil_div(p.tb, p.slices), kColStep);
        p.slices = ceil_div(p.tb, p.slice);
        p.tail_pairs = rest * p.slices;
    } else {
        long long shares = static_cast<long long>(rest) * p.kc / kMinChunks;
        if (shares > p.pairs) shares = p.pairs;
        if (shares < rest) shares = rest;
        p.slice = p.tb;
        p.tail_pairs = static_cast<int>(shares);
    }
    if (p.full == 0) p.pairs = p.tail_pairs;
    p.width = p.full == 0 && p.slices > 0 ? p.slice : p.tb;
    p.stage_bytes = kGroup * (kRows + p.width / 2) * 128;
    p.stages = kSmemCap / p.stage_bytes;
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    p.ksplit = 1;
    while (p.ksplit < 8 && K >= 32 * kShrinkWarps * 2 * p.ksplit) p.ksplit *= 2;
    // as many shrink clusters as have work, at most two CTAs per SM: they share a token block's units or
    // walk the blocks
    const int most = (p.slots < M ? p.slots : M) + (M < p.tb ? M : p.tb) / kShrinkTok;   // units of a block
    const int qs = ceil_div(p.rsteps, shrink_steps(p.rsteps));
    const int fit = 2 * sms / p.ksplit;
    p.per_blk = fit / p.nb < 1 ? 1 : fit / p.nb < most * qs ? fit / p.nb : most * qs;
    p.clusters = p.per_blk * (fit / p.per_blk < p.nb ? fit / p.per_blk : p.nb);
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off = (off + bytes + 255) / 256 * 256;
        return at;
    };
    p.off_status = take(256);
    p.off_count = take(sizeof(int) * 2 * kJoins * static_cast<size_t>(p.pairs));
    p.off_meta = take(sizeof(int2) * static_cast<size_t>(p.nb) * (p.slots + 1));
    p.off_perm = take(sizeof(int) * kMaxTok);
    p.off_x = take(p.sorted ? static_cast<size_t>(p.tb) * K * 2 : 0);
    p.off_u = take(static_cast<size_t>(p.nb) * p.slots * p.rchunks * p.tb * p.kw * 2);
    p.off_u32 = take(static_cast<size_t>(p.nb) * p.tb * p.rsteps * kStep * sizeof(float));
    p.off_part = take(p.slices == 0 && p.tail_pairs > rest ? static_cast<size_t>(p.tail_pairs) * 4 * kRows * p.tb * sizeof(float) : 0);
    p.total = off;
    return p;
}

// An adapter of a token block: its id, its place in the block's list, the first of its tokens' columns
// and how many an MMA covers (both multiples of 32).
__device__ __forceinline__ int2 pack_slot(int id, int slot, int lo, int n) {
    return make_int2(id, slot << 16 | lo / kColStep << 8 | n / kColStep);
}
__device__ __forceinline__ int slot_of(int2 s) { return s.y >> 16; }
__device__ __forceinline__ int slot_lo(int2 s) { return (s.y >> 8 & 255) * kColStep; }
__device__ __forceinline__ int slot_n(int2 s) { return (s.y & 255) * kColStep; }

template <typename T>
__device__ __forceinline__ void to_float8(const uint4& v, float (&f)[8]) {
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = ElemTraits<T>::to_f2(*reinterpret_cast<const typename ElemTraits<T>::T2*>(&x[i]));
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}
// U in fp32, of the token in a block's column.
__device__ __forceinline__ float* u32_row(const Plan& P, unsigned char* ws, int blk, int col) {
    return reinterpret_cast<float*>(ws + P.off_u32) + (static_cast<size_t>(blk) * P.tb + col) * P.rsteps * kStep;
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

// The tokens of a block by adapter.
struct Order {
    int ids[kMaxTok];                       // adapter, or -1
    short col_of[kMaxTok], tok_of[kMaxTok]; // a token's column, and back (-1)
    // of an adapter, at its first token: first column in adapter order, slot, first unit, columns an MMA covers
    short base[kMaxTok], slot[kMaxTok], unit0[kMaxTok];
    short2 cover[kMaxTok];
    short unit_lead[kMaxTok + kMaxTok / kShrinkTok];   // a unit's adapter, as its first token
    int warp_sum[kShrinkWarps];
    int slots, units;
};
// Per adapter while the tokens are counted: tokens so far, first, last.
struct Table {
    short n[kTable], first[kTable], last[kTable];
};
struct Own {
    int id, first, rank_in;               // this thread's token: adapter, the adapter's first token, place among its tokens
};

// Sorts block blk's tokens by adapter (stable), one thread a token. Adapters follow the order of their
// first tokens; tokens without one come last.
__device__ __forceinline__ Own order_tokens(Order& o, Table& tab, const LoraArgs& A, const Plan& P, int blk) {
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int m0 = blk * P.tb, mt = min(P.tb, P.M - m0);
    __syncthreads();   // (the block before has been read)
    const int raw = tid < mt ? A.ids[m0 + tid] : -1, id = raw >= 0 && raw < P.adapters ? raw : -1;
    o.ids[tid] = id;
    o.tok_of[tid] = -1;
    int count = 0, rank_in = 0, first = kMaxTok, last = 0;
    if (P.adapters <= kTable) {
        // one warp after the other enters its tokens, 32 at a time matched among each other
        for (int i = tid; i < P.adapters; i += blockDim.x) tab.n[i] = 0;
        __syncthreads();
        const unsigned same = __match_any_sync(0xffffffffu, id), less = (1u << lane) - 1;
        for (int w = 0; w < kShrinkWarps && w * 32 < mt; ++w) {
            if (w == warp) {
                if (id >= 0) rank_in = tab.n[id] + __popc(same & less);
                __syncwarp();
                if (id >= 0 && lane == 31 - __clz(same)) {
                    if (rank_in + 1 == __popc(same)) tab.first[id] = static_cast<short>(warp * 32 + __ffs(same) - 1);
                    tab.n[id] = static_cast<short>(rank_in + 1);
                    tab.last[id] = static_cast<short>(tid);
                }
            }
            __syncthreads();
        }
        if (id >= 0) {
            count = tab.n[id];
            first = tab.first[id];
            last = tab.last[id];
        }
    } else {
        __syncthreads();
        for (int j = 0; j < mt; ++j)
            if (o.ids[j] == id && id >= 0) {
                if (count == 0) first = j;
                last = j;
                rank_in += j < tid;
                ++count;
            }
    }
    const unsigned none = __ballot_sync(0xffffffffu, id < 0);
    if (lane == 0) o.warp_sum[warp] = __popc(none);
    __syncthreads();
    if (id < 0) {
        rank_in = __popc(none & ((1u << lane) - 1));
        for (int w = 0; w < warp; ++w) rank_in += o.warp_sum[w];
    }
    __syncthreads();
    const bool leader = id >= 0 && first == tid;
    const int groups = leader ? (count + kShrinkTok - 1) / kShrinkTok : 0;
    // sums over the leaders before: adapters, units, tokens (each below 1024)
    const int v = leader ? 1 | groups << 10 | count << 20 : 0;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += a;
    }
    if (lane == 31) o.warp_sum[warp] = x;
    __syncthreads();
    int total = 0, before = x - v;
    for (int w = 0; w < kShrinkWarps; ++w) {
        if (w < warp) before += o.warp_sum[w];
        total += o.warp_sum[w];
    }
    if (leader) {
        const int u0 = before >> 10 & 1023, b0 = before >> 20;
        o.base[tid] = static_cast<short>(b0);
        o.slot[tid] = static_cast<short>(before & 1023);
        o.unit0[tid] = static_cast<short>(u0);
        for (int i = 0; i < groups; ++i) o.unit_lead[u0 + i] = static_cast<short>(tid);
        // the columns an MMA covers: the adapter's tokens (all between its first and its last where the
        // block is not sorted), from a multiple of 32 (where an accumulator may begin) to one
        const int c0 = P.sorted ? b0 : first, c1 = P.sorted ? b0 + count : last + 1;
        const int lo = c0 / kColStep * kColStep;
        o.cover[tid] = make_short2(static_cast<short>(lo), static_cast<short>((c1 - lo + kColStep - 1) / kColStep * kColStep));
    }
    if (tid == 0) {
        o.slots = total & 1023;
        o.units = total >> 10 & 1023;
    }
    __syncthreads();
    if (tid < mt) {
        const int c = !P.sorted ? tid : id >= 0 ? o.base[first] + rank_in : (total >> 20) + rank_in;
        o.col_of[tid] = static_cast<short>(c);
        o.tok_of[c] = static_cast<short>(tid);
    }
    __syncthreads();
    return {id, first, rank_in};
}

// Clusters of ksplit CTAs, which cut K, walk items of one unit and kQ rank steps: a unit is one adapter
// of a token block with up to 32 of its tokens. Each of a CTA's warps takes every (8 ksplit)-th 32
// columns of K and holds the 16 kQ ranks x 32 tokens in registers as warp-level MMA tiles, reading A's
// and x's rows straight from global memory, 16 bytes a lane: the sum over K may take its columns in any
// order, so lane t of a quad takes columns 8 t .. 8 t + 7 of each 32, for both operands alike. Tokens
// are gathered by their rows' addresses. Partial sums meet in shared memory, in warp order and then in
// CTA order. (16 ranks x 32 tokens are too small for tcgen05's 128-row tile. Letting the GEMM run beside
// it, with registers left for both, was slower: its few loads in flight wait behind the GEMM's, 108 us
// instead of 23 for 256 tokens with 32 adapters of rank 64 over K = 7168.)
template <typename T, int kQ>
__global__ void __launch_bounds__(32 * kShrinkWarps, 2) lora_shrink_kernel(const LoraArgs A, const Plan P, unsigned char* ws) {
    __shared__ Order o;
    __shared__ int list[kShrinkTok];
    __shared__ union {
        Table tab;
        float red[kShrinkWarps][kStep][kShrinkTok + 1];   // the warps' partial sums
    } sh;
    __shared__ float part[kQ][kStep][kShrinkTok];         // this CTA's sums
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int cluster = blockIdx.x / P.ksplit, kpart = blockIdx.x % P.ksplit;
    if (blockIdx.x == 0) {
        int* count = reinterpret_cast<int*>(ws + P.off_count);
        for (int i = tid; i < 2 * kJoins * P.pairs; i += blockDim.x) count[i] = 0;
        if (tid == 0) *reinterpret_cast<int*>(ws + P.off_status) = 0;
    }
    const int qsteps = (P.rsteps + kQ - 1) / kQ;
    for (int blk = cluster / P.per_blk; blk < P.nb; blk += P.clusters / P.per_blk) {
        const int m0 = blk * P.tb;
        const Own own = order_tokens(o, sh.tab, A, P, blk);
        if (cluster % P.per_blk == 0 && kpart == 0) {
            int2* meta = reinterpret_cast<int2*>(ws + P.off_meta) + static_cast<size_t>(blk) * (P.slots + 1);
            if (own.id >= 0 && own.first == tid) meta[1 + o.slot[tid]] = pack_slot(own.id, o.slot[tid], o.cover[tid].x, o.cover[tid].y);
            if (tid == 0) meta[0] = make_int2(o.slots, 0);
        }
        if (P.sorted) {
            // X's rows in adapter order, and the order; the CTAs take the columns in turn
            const int nvec = P.K / 8;
            if (blockIdx.x == 0 && tid < P.M) reinterpret_cast<int*>(ws + P.off_perm)[tid] = o.tok_of[tid];
            for (int c = blockIdx.x; c < P.M; c += gridDim.x) {
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(A.x) + static_cast<long long>(o.tok_of[c]) * A.x_stride);
                uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(ws + P.off_x) + static_cast<size_t>(c) * P.K);
#pragma unroll 4
                for (int i = tid; i < nvec; i += blockDim.x) dst[i] = __ldg(src + i);
            }
        }
        for (int item = cluster % P.per_blk; item < o.units * qsteps; item += P.per_blk) {
            const int lead = o.unit_lead[item / qsteps], sub = item / qsteps - o.unit0[lead], q0 = item % qsteps * kQ;
            const int a = o.ids[lead], unit_slot = o.slot[lead], unit_lo = o.cover[lead].x, unit_n = o.cover[lead].y;
            if (tid < kShrinkTok) list[tid] = -1;
            __syncthreads();
            if (own.id == a && own.rank_in / kShrinkTok == sub) list[own.rank_in % kShrinkTok] = tid;
            __syncthreads();
            const int g = lane / 4, t = lane % 4;
            const T* arow = static_cast<const T*>(A.a) + (static_cast<long long>(a) * P.r + q0 * kStep + g) * P.K;
            const int left = P.r - q0 * kStep - g;   // ranks from this lane's first on
            const T* xrow[4];
            int nt = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int m = list[8 * i + g];
                xrow[i] = m >= 0 ? static_cast<const T*>(A.x) + (m0 + m) * A.x_stride : nullptr;
                if (list[8 * i] >= 0) nt = i + 1;
            }
            float acc[kQ][4][4] = {};
            constexpr int kUnroll = 4 / kQ;
            const int stride = 32 * kShrinkWarps * P.ksplit;
            for (int k0 = 32 * (kpart * kShrinkWarps + warp); k0 < P.K; k0 += stride * kUnroll) {
                uint4 va[kUnroll][kQ][2], vx[kUnroll][4];
#pragma unroll
                for (int j = 0; j < kUnroll; ++j) {
                    const int k = k0 + j * stride + 8 * t;
#pragma unroll
                    for (int e = 0; e < kQ; ++e)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            va[j][e][i] = e * kStep + 8 * i < left && k < P.K
                                              ? __ldg(reinterpret_cast<const uint4*>(arow + (e * kStep + 8 * i) * static_cast<long long>(P.K) + k))
                                              : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        vx[j][i] = xrow[i] && k < P.K ? __ldg(reinterpret_cast<const uint4*>(xrow[i] + k)) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < kUnroll; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i < nt)
#pragma unroll
                            for (int e = 0; e < kQ; ++e) {
                                const uint4 r0 = va[j][e][0], r1 = va[j][e][1], v = vx[j][i];
                                mma16816<T>(acc[e][i], r0.x, r1.x, r0.y, r1.y, v.x, v.y);
                                mma16816<T>(acc[e][i], r0.z, r1.z, r0.w, r1.w, v.z, v.w);
                            }
            }
#pragma unroll
            for (int e = 0; e < kQ; ++e) {
                __syncthreads();   // (the step before has been read)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sh.red[warp][g][8 * i + 2 * t] = acc[e][i][0];
                    sh.red[warp][g][8 * i + 2 * t + 1] = acc[e][i][1];
                    sh.red[warp][g + 8][8 * i + 2 * t] = acc[e][i][2];
                    sh.red[warp][g + 8][8 * i + 2 * t + 1] = acc[e][i][3];
                }
                __syncthreads();
                for (int i = tid; i < kStep * kShrinkTok; i += blockDim.x) {
                    float s = 0.f;
#pragma unroll
                    for (int w = 0; w < kShrinkWarps; ++w) s += sh.red[w][i / kShrinkTok][i % kShrinkTok];
                    part[e][i / kShrinkTok][i % kShrinkTok] = s;
                }
            }
            if (P.ksplit > 1) cluster_sync();
            else __syncthreads();
            // the adapter's U rows: its tokens' values, zeros in the other columns that the MMA covers; the
            // cluster's CTAs take the tokens in turn
            const float scale = A.scales ? A.scales[a] : 1.f;
#pragma unroll
            for (int e = 0; e < kQ; ++e) {
                if (q0 + e >= P.rsteps) break;
                const int spc = P.kw / kStep, q = q0 + e;
                T* u = reinterpret_cast<T*>(ws + P.off_u) + q % spc * kStep +
                       ((static_cast<size_t>(blk) * P.slots + unit_slot) * P.rchunks + q / spc) * P.tb * P.kw;
                for (int i = tid + kpart * blockDim.x; i < kStep * kShrinkTok; i += blockDim.x * P.ksplit) {
                    const int k = i % kStep, j = i / kStep, m = list[j];
                    if (m < 0) continue;
                    const uint32_t at = smem_u32(&part[e][k][j]);
                    float s = 0.f;
                    for (int c = 0; c < P.ksplit; ++c) {
                        float y;
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y) : "r"(mapa(at, c)));
                        s += y;
                    }
                    u[o.col_of[m] * P.kw + k] = ElemTraits<T>::from_f(s * scale);
                    u32_row(P, ws, blk, o.col_of[m])[q * kStep + k] = s * scale;
                }
                if (sub == 0 && kpart == P.ksplit - 1)
                    for (int i = tid; i < unit_n * 2; i += blockDim.x) {
                        const int c = unit_lo + i / 2, m = o.tok_of[c];
                        if (m < 0 || o.ids[m] != a) *reinterpret_cast<uint4*>(u + c * P.kw + i % 2 * 8) = make_uint4(0, 0, 0, 0);
                    }
            }
            if (P.ksplit > 1) cluster_sync();   // no CTA leaves or goes on while its sums may be read
            else __syncthreads();
        }
    }
}

// ------------------------------------------------------------------------------------- GEMM

struct Maps {
    CUtensorMap w, x, xs, b, u;
};

// One piece of a pair's work: chunks [c0, c1) of K and columns [lo, lo + cols) of a tile.
struct Item {
    int tile, c0, c1;
    int lo, cols;
    int j;           // index among the tiles cut along K, or -1
};
// Walks the pair's pieces; every role walks an identical copy.
struct Walk {
    int next_full, slice;
    long long c, c_end;
    __device__ explicit Walk(const Plan& P) {
        const int w = blockIdx.x / 2;
        next_full = w;
        c = c_end = 0;
        slice = P.slices > 0 && w < P.tail_pairs ? w : -1;
        if (P.slices == 0 && w < P.tail_pairs) {
            const long long total = static_cast<long long>(P.tiles - P.full) * P.kc;
            c = total * w / P.tail_pairs;
            c_end = total * (w + 1) / P.tail_pairs;
        }
    }
    // columns of a tile's block: its tokens, up to a multiple of 32
    static __device__ int block_cols(const Plan& P, int tile) {
        return (min(P.tb, P.M - tile % P.nb * P.tb) + kColStep - 1) / kColStep * kColStep;
    }
    __device__ bool next(const Plan& P, Item* it) {
        if (next_full < P.full) {
            *it = {next_full, 0, P.kc, 0, block_cols(P, next_full), -1};
            next_full += P.pairs;
            return true;
        }
        if (slice >= 0) {
            const int tile = P.full + slice / P.slices, lo = slice % P.slices * P.slice;
            const int cols = min(P.slice, block_cols(P, tile) - lo);
            slice = -1;
            *it = {tile, 0, P.kc, lo, cols, -1};
            return cols > 0;
        }
        if (c >= c_end) return false;
        const int j = static_cast<int>(c / P.kc);
        const int c0 = static_cast<int>(c % P.kc);
        const int n = static_cast<int>(c_end - c);
        const int c1 = min(P.kc, c0 + n);
        *it = {P.full + j, c0, c1, 0, block_cols(P, P.full + j), j};
        c += c1 - c0;
        return true;
    }
};

struct __align__(16) Bars {
    uint64_t full[kMaxStages];        // leader: both CTAs' loads of the stage have landed
    uint64_t empty[kMaxStages];       // both: the MMAs have read it
    uint64_t acc_full[2];             // both: the accumulator is complete
    uint64_t acc_empty[2];            // leader: both CTAs have read it out
    uint32_t tmem;
    int last;
    __align__(16) int perm[kMaxTok];  // output row of each column (sorted)
    int2 slots[2][kMaxTok];           // the block's adapters, for the loading and the issuing warp
};

static_assert(offsetof(Bars, perm) % 16 == 0, "read as int4");

__device__ __forceinline__ int code(int site) { return kStatusTimeout | (site << 8); }

// K-major tile whose rows hold kw ranks, swizzled to its row length
__device__ __forceinline__ uint64_t rank_desc(uint32_t addr, int kw) {
    return kw == 64 ? smem_desc_sw128(addr, 16, 1024) : kw == 32 ? smem_desc_sw64(addr) : smem_desc_sw32(addr);
}

// The adapters of token block blk that have columns of [lo, lo + cols) into sl (one warp), their columns
// from lo on; returns how many.
__device__ __forceinline__ int load_slots(const Plan& P, const unsigned char* ws, int blk, int lo, int cols, int2* sl, int lane) {
    const int2* meta = reinterpret_cast<const int2*>(ws + P.off_meta) + static_cast<size_t>(blk) * (P.slots + 1);
    const int n = meta[0].x;
    int kept = 0;
    __syncwarp();
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int2 s = i0 + lane < n ? meta[1 + i0 + lane] : make_int2(0, 0);
        const int a = max(slot_lo(s), lo), b = min(slot_lo(s) + slot_n(s), lo + cols);
        const unsigned in = __ballot_sync(0xffffffffu, i0 + lane < n && a < b);
        if (in >> lane & 1) sl[kept + __popc(in & ((1u << lane) - 1))] = pack_slot(s.x, slot_of(s), a - lo, b - a);
        kept += __popc(in);
    }
    __syncwarp();
    return kept;
}

// The infinite and NaN outputs among sixteen columns of a warp's 32 weight rows (lane = row n0 + lane) from the
// tokens' own operands, U in fp32: the rare path of outputs that another token's adapter broke, or U where it
// passed the type's range. perm: the columns' tokens where they are sorted. An output that its own adapter makes
// NaN stays one; for the others W x is computed again, for the warp's rows and the columns at once, on
// warp-level MMAs. (One NaN adapter of 12 in a batch of 67 tokens: 1.1 ms, element by element 153.) It works on
// the outputs as they were stored, after all read-outs: called from there, it cost them registers (the same
// batch without NaN 70 -> 75 us).
template <typename T>
__device__ __noinline__ void own_columns(const LoraArgs& A, const Plan& P, unsigned char* ws, int blk, int c, int n0, int toks,
                                         const int* perm) {
    const int lane = threadIdx.x & 31, n = n0 + lane;
    auto tok = [&](int k) { return P.sorted ? perm[c + k] : blk * P.tb + c + k; };
    T* y = static_cast<T*>(A.y) + n;
    uint32_t need = 0;
    float w[16];   // the adapters' parts
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        w[k] = 0.f;
        if (n < P.N && c + k < toks && !isfinite(ElemTraits<T>::to_f(y[static_cast<long long>(tok(k)) * P.N]))) {
            const int id = A.ids[tok(k)];
            float v = 0.f;
            if (id >= 0 && id < P.adapters) {
                const float* u = u32_row(P, ws, blk, c + k);
                const uint4* b = reinterpret_cast<const uint4*>(static_cast<const T*>(A.b) + (static_cast<long long>(id) * P.N + n) * P.r);
                for (int i = 0; i < P.r; i += 8) {
                    float f[8];
                    to_float8<T>(b[i / 8], f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v = fmaf(u[i + e], f[e], v);
                }
            }
            w[k] = v;
            if (v == v) need |= 1u << k;
        }
    }
    if (!__any_sync(0xffffffffu, need != 0)) return;
    // W x: a quad's lane t takes columns 8 t .. 8 t + 7 of each 32 of K, for both operands alike
    const int g = lane / 4, t = lane % 4;
    const T *wr[4], *xr[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) wr[i] = static_cast<const T*>(A.w) + static_cast<long long>(min(n0 + 8 * i + g, P.N - 1)) * P.K + 8 * t;
#pragma unroll
    for (int i = 0; i < 2; ++i) xr[i] = static_cast<const T*>(A.x) + static_cast<long long>(tok(min(8 * i + g, toks - c - 1))) * A.x_stride + 8 * t;
    float acc[2][2][4] = {};
    constexpr int kAhead = 4;
    for (int k0 = 0; k0 < P.K; k0 += 32 * kAhead) {
        uint4 vw[kAhead][4], vx[kAhead][2];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int k = k0 + 32 * j;
            const bool in = k + 8 * t < P.K;
#pragma unroll
            for (int i = 0; i < 4; ++i) vw[j][i] = in ? __ldg(reinterpret_cast<const uint4*>(wr[i] + k)) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 2; ++i) vx[j][i] = in ? __ldg(reinterpret_cast<const uint4*>(xr[i] + k)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 r0 = vw[j][2 * m], r1 = vw[j][2 * m + 1], v = vx[j][i];
                    mma16816<T>(acc[m][i], r0.x, r1.x, r0.y, r1.y, v.x, v.y);
                    mma16816<T>(acc[m][i], r0.z, r1.z, r0.w, r1.w, v.z, v.w);
                }
    }
    // row 16 m + 8 h + g', column 8 i + 2 t' + e of the product is at lane 4 g' + t', acc[m][i][2 h + e]
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int src = lane % 8 * 4 + k % 8 / 2;
        float z[4];   // by (m, h)
#pragma unroll
        for (int q = 0; q < 4; ++q) z[q] = __shfl_sync(0xffffffffu, acc[q / 2][k / 8][2 * (q % 2) + k % 2], src);
        const float v = w[k] + (lane & 16 ? (lane & 8 ? z[3] : z[2]) : (lane & 8 ? z[1] : z[0]));
        if (need >> k & 1) y[static_cast<long long>(tok(k)) * P.N] = ElemTraits<T>::from_f(v);
    }
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
lora_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Plan P,
                 const __grid_constant__ LoraArgs A, unsigned char* ws) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Bars* bars = reinterpret_cast<Bars*>(smem + P.stages * P.stage_bytes);
    const uint32_t ring = smem_u32(smem);
    const uint32_t rank = cluster_ctarank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* err = reinterpret_cast<int*>(ws + P.off_status);
    // a stage: W chunks (then the adapters' B rows) | X chunks (then U rows)
    const uint32_t x_off = kGroup * kRows * 128, x_chunk = P.width / 2 * 128;
    const uint32_t b_chunk = kRows * P.kw * 2, u_chunk = P.width / 2 * P.kw * 2;
    const int per_stage = kGroup * kChunk / P.kw;   // of B's and U's tiles
    if (threadIdx.x == 0) {
        for (int s = 0; s < P.stages; ++s) {
            mbar_init(smem_u32(&bars->full[s]), 1);
            mbar_init(smem_u32(&bars->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&bars->acc_full[b]), 1);
            mbar_init(smem_u32(&bars->acc_empty[b]), 8);   // one arrival per reading warp of the pair
        }
        fence_mbar_init();
        tma_prefetch_desc(&maps.w);
        tma_prefetch_desc(&maps.x);
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(&bars->tmem), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tbase = bars->tmem;

    if (warp == 0) {
        // ---- loads: this CTA's weight rows and half of the tokens' rows
        // (this and the issuing warp start before the shrink kernel has cleared the status word: their waits
        // end on completion or on their own limit and do not look at it)
        Walk walk(P);
        Item it;
        int i = 0, blk_slots = -1, lo_slots = -1, cols_slots = -1, nslots = 0;
        bool ok = true, waited = !P.sorted;   // X in adapter order comes from the shrink kernel
        bool meta_ready = false;
        int held = 0;                         // stages whose W is on its way while X is waited for
        while (ok && walk.next(P, &it)) {
            const int n0 = it.tile / P.nb * 2 * kRows + static_cast<int>(rank) * kRows, blk = it.tile % P.nb;
            const int x0 = (P.sorted ? 0 : blk * P.tb) + it.lo + static_cast<int>(rank) * it.cols / 2;   // this CTA's half
            // (boxes of half a block's or half a slice's rows; only the columns of the piece are used)
            const bool cut = P.slices > 0 && it.tile >= P.full;
            const CUtensorMap* xmap = cut ? &maps.xs : &maps.x;
            const uint32_t x_bytes = cut ? P.slice / 2 * 128 : x_chunk;
            for (int c = it.c0; c < it.c1; c += kGroup, ++i) {
                const int s = i % P.stages;
                ok = i < P.stages || mbar_wait_cluster_full(smem_u32(&bars->empty[s]), ((i / P.stages) - 1) & 1, err, code(kWaitLoad));
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                const int n = min(kGroup, it.c1 - c);
                const uint32_t fb = mapa(smem_u32(&bars->full[s]), 0), dst = ring + s * P.stage_bytes;
                if (elect_one()) {
                    if (rank == 0)
                        mbar_arrive_expect_tx(smem_u32(&bars->full[s]), 2u * n * (kRows * 128 + x_bytes));
                    for (int k = 0; k < n; ++k)
                        tma_load_2d_pair(dst + k * kRows * 128, &maps.w, fb, kChunk * (c + k), n0);
                    if (waited)
                        for (int k = 0; k < n; ++k)
                            tma_load_2d_pair(dst + x_off + k * x_chunk, xmap, fb, kChunk * (c + k), x0);
                }
                __syncwarp();
                if (!waited) {
                    // W of the first stages streams in while the shrink kernel puts X in order
                    ++held;
                    if (held == P.stages || c + kGroup >= it.c1) {
                        pdl_wait();
                        waited = meta_ready = true;
                        if (elect_one())
                            for (int h = 0; h < held; ++h) {
                                const int hc = c - (held - 1 - h) * kGroup, hs = i - (held - 1 - h);
                                const uint32_t hb = mapa(smem_u32(&bars->full[hs % P.stages]), 0);
                                for (int k = 0; k < min(kGroup, it.c1 - hc); ++k)
                                    tma_load_2d_pair(ring + (hs % P.stages) * P.stage_bytes + x_off + k * x_chunk, xmap, hb,
                                                     kChunk * (hc + k), x0);
                            }
                        __syncwarp();
                    }
                }
            }
            if (!ok || it.c1 < P.kc) continue;
            if (!meta_ready) {
                pdl_wait();   // U and the adapters' list come from the shrink kernel
                meta_ready = true;
            }
            if (blk != blk_slots || it.lo != lo_slots || it.cols != cols_slots)
                nslots = load_slots(P, ws, blk, it.lo, it.cols, bars->slots[0], lane);
            blk_slots = blk;
            lo_slots = it.lo;
            cols_slots = it.cols;
            const int chunks = nslots * P.rchunks;
            for (int s0 = 0; s0 < chunks; s0 += per_stage, ++i) {
                const int s = i % P.stages;
                ok = i < P.stages || mbar_wait_cluster_full(smem_u32(&bars->empty[s]), ((i / P.stages) - 1) & 1, err, code(kWaitLoad));
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                const int n = min(per_stage, chunks - s0);
                if (elect_one()) {
                    const uint32_t fb = mapa(smem_u32(&bars->full[s]), 0), dst = ring + s * P.stage_bytes;
                    if (rank == 0) {
                        uint32_t bytes = 2u * n * b_chunk;
                        for (int k = 0; k < n; ++k) bytes += slot_n(bars->slots[0][(s0 + k) / P.rchunks]) * P.kw * 2;
                        mbar_arrive_expect_tx(smem_u32(&bars->full[s]), bytes);
                    }
                    for (int k = 0; k < n; ++k) {
                        const int2 sl = bars->slots[0][(s0 + k) / P.rchunks];
                        const int q = (s0 + k) % P.rchunks, half_n = slot_n(sl) / 2;
                        tma_load_3d_pair(dst + k * b_chunk, &maps.b, fb, q * P.kw, n0, sl.x);
                        const int u0 = ((blk * P.slots + slot_of(sl)) * P.rchunks + q) * P.tb + it.lo + slot_lo(sl) +
                                       static_cast<int>(rank) * half_n;
                        for (int c = 0; c < half_n; c += kColStep / 2)
                            tma_load_2d_pair(dst + x_off + k * u_chunk + c * P.kw * 2, &maps.u, fb, 0, u0 + c);
                    }
                }
                __syncwarp();
            }
        }
        if (!meta_ready) pdl_wait();
    } else if (warp == 1) {
        // ---- MMAs of the pair
        if (rank == 0) {
            Walk walk(P);
            Item it;
            int i = 0, n = 0, blk_slots = -1, lo_slots = -1, cols_slots = -1, nslots = 0;
            bool ok = true, meta_ready = false;
            for (; ok && walk.next(P, &it); ++n) {
                const int blk = it.tile % P.nb;
                const uint32_t idesc = idesc_f16(256, it.cols, Fmt<T>::v, false, false);
                const uint32_t d = tbase + 256 * (n & 1);
                ok = n < 2 || mbar_wait_cluster_full(smem_u32(&bars->acc_empty[n & 1]), ((n >> 1) - 1) & 1, err, code(kWaitAcc));
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                for (int c = it.c0; c < it.c1; c += kGroup, ++i) {
                    const int s = i % P.stages;
                    ok = mbar_wait_cluster_full(smem_u32(&bars->full[s]), (i / P.stages) & 1, err, code(kWaitMma));
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t a = ring + s * P.stage_bytes;
                        for (int k = 0; k < min(kGroup, it.c1 - c); ++k) {
                            const uint64_t ad = smem_desc_sw128(a + k * kRows * 128, 16, 1024);
                            const uint64_t bd = smem_desc_sw128(a + x_off + k * x_chunk, 16, 1024);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                mma_ss_pair(d, ad + static_cast<uint64_t>(2 * e), bd + static_cast<uint64_t>(2 * e), idesc,
                                            c + k > it.c0 || e > 0 ? 1u : 0u);
                        }
                        mma_commit_pair_both(smem_u32(&bars->empty[s]));
                    }
                    __syncwarp();
                }
                if (ok && it.c1 == P.kc) {
                    if (!meta_ready) {
                        pdl_wait();
                        meta_ready = true;
                    }
                    if (blk != blk_slots || it.lo != lo_slots || it.cols != cols_slots)
                        nslots = load_slots(P, ws, blk, it.lo, it.cols, bars->slots[1], lane);
                    blk_slots = blk;
                    lo_slots = it.lo;
                    cols_slots = it.cols;
                    const int chunks = nslots * P.rchunks;
                    for (int s0 = 0; s0 < chunks; s0 += per_stage, ++i) {
                        const int s = i % P.stages;
                        ok = mbar_wait_cluster_full(smem_u32(&bars->full[s]), (i / P.stages) & 1, err, code(kWaitMma));
                        if (!__all_sync(0xffffffffu, ok)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t a = ring + s * P.stage_bytes;
                            for (int k = 0; k < min(per_stage, chunks - s0); ++k) {
                                const int2 sl = bars->slots[1][(s0 + k) / P.rchunks];
                                const int steps = min(P.kw / kStep, P.rsteps - (s0 + k) % P.rchunks * (P.kw / kStep));
                                const uint64_t ad = rank_desc(a + k * b_chunk, P.kw), bd = rank_desc(a + x_off + k * u_chunk, P.kw);
                                const uint32_t id = idesc_f16(256, slot_n(sl), Fmt<T>::v, false, false);
                                for (int e = 0; e < steps; ++e)
                                    mma_ss_pair(d + slot_lo(sl), ad + static_cast<uint64_t>(2 * e), bd + static_cast<uint64_t>(2 * e), id, 1u);
                            }
                            mma_commit_pair_both(smem_u32(&bars->empty[s]));
                        }
                        __syncwarp();
                    }
                }
                if (elect_one()) mma_commit_pair_both(smem_u32(&bars->acc_full[n & 1]));
                __syncwarp();
            }
        }
    } else {
        // ---- read-out: thread = weight row = TMEM lane
        const int row = (warp & 3) * 32 + lane;
        const uint32_t trow = tbase + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
        const uint32_t acc_empty0 = mapa(smem_u32(&bars->acc_empty[0]), 0), acc_empty1 = mapa(smem_u32(&bars->acc_empty[1]), 0);
        Walk walk(P);
        Item it;
        bool ok = true, broken = false;   // (a broken output of this thread's)
        // of the tiles cut along K, at most two: the columns that this CTA stored, in kJoinCols
        uint32_t joined = 0;
        auto joined_at = [&](int j) {
            const long long c0 = static_cast<long long>(P.tiles - P.full) * P.kc * (blockIdx.x / 2) / P.tail_pairs;
            return c0 / P.kc == j ? 0 : kJoins;
        };
        pdl_wait();   // the counters are cleared and the columns' order is written by the shrink kernel
        if (P.sorted)
            for (int c = threadIdx.x - 64; c < P.M; c += 128) bars->perm[c] = reinterpret_cast<const int*>(ws + P.off_perm)[c];
        asm volatile("bar.sync 1, 128;" ::: "memory");
        for (int n = 0; walk.next(P, &it); ++n) {
            const int blk = it.tile % P.nb, m0 = blk * P.tb, toks = min(P.tb, P.M - m0);
            const int col = it.tile / P.nb * 2 * kRows + static_cast<int>(rank) * kRows + row;
            const uint32_t d = trow + 256 * (n & 1);
            const bool got = mbar_wait_cluster(smem_u32(&bars->acc_full[n & 1]), (n >> 1) & 1, err, code(kWaitOut));
            ok = __all_sync(0xffffffffu, got) && ok;
            tc_fence_after();
            const bool any = reinterpret_cast<const int2*>(ws + P.off_meta)[static_cast<size_t>(blk) * (P.slots + 1)].x > 0;
            // 16 columns from c on of this thread's weight row
            auto store16 = [&](int c, const float* v) {
                int m[16];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int4 w = P.sorted ? *reinterpret_cast<const int4*>(bars->perm + c + 4 * k)
                                            : make_int4(m0 + c + 4 * k, m0 + c + 4 * k + 1, m0 + c + 4 * k + 2, m0 + c + 4 * k + 3);
                    m[4 * k] = w.x;
                    m[4 * k + 1] = w.y;
                    m[4 * k + 2] = w.z;
                    m[4 * k + 3] = w.w;
                }
                bool finite = true;
#pragma unroll
                for (int k = 0; k < 16; ++k) finite = finite && isfinite(v[k]);
                T* y = static_cast<T*>(A.y) + col;
                broken = broken || (!finite && any && ok && col < P.N);
                if (col >= P.N) return;
                if (c + 16 <= toks && ok) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) y[static_cast<long long>(m[k]) * P.N] = ElemTraits<T>::from_f(v[k]);
                    return;
                }
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (c + k < toks) y[static_cast<long long>(m[k]) * P.N] = ElemTraits<T>::from_f(ok ? v[k] : NAN);
            };
            auto release = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (rank == 0) mbar_arrive(smem_u32(&bars->acc_empty[n & 1]));
                    else mbar_arrive_remote(n & 1 ? acc_empty1 : acc_empty0);
                }
            };
            // the pairs that share the tile
            int w0 = blockIdx.x / 2, w1 = w0;
            const long long total = static_cast<long long>(P.tiles - P.full) * P.kc;
            if (it.j >= 0) {
                w0 = static_cast<int>(((static_cast<long long>(it.j) * P.kc + 1) * P.tail_pairs - 1) / total);
                w1 = static_cast<int>(((static_cast<long long>(it.j) + 1) * P.kc * P.tail_pairs - 1) / total);
            }
            if (w0 == w1) {
                if (it.j >= 0) joined |= ((1u << kJoins) - 1) << joined_at(it.j);
                for (int c = 0; c < min(it.cols, toks - it.lo); c += 16) {
                    uint32_t u[16];
                    tmem_ld16_sync(d + c, u);
                    float v[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) v[k] = __uint_as_float(u[k]);
                    store16(it.lo + c, v);
                }
            } else {
                // partials as float4 of 4 columns: column group g of row r at g * kRows + r
                float4* parts = reinterpret_cast<float4*>(ws + P.off_part);
                auto part = [&](int w) -> float4* {
                    // a pair touches at most two cut tiles: the first into its place 0, the second into place 1
                    const int first = static_cast<int>(total * w / P.tail_pairs / P.kc);
                    return parts + ((static_cast<size_t>(w) * 2 + (first == it.j ? 0 : 1)) * 2 + rank) * kRows * P.tb / 4 + row;
                };
                const int me = blockIdx.x / 2, joins = (toks + kJoinCols - 1) / kJoinCols;
                float4* mine = part(me);
                for (int c = 0; c < toks; c += 16) {
                    uint32_t v[16];
                    tmem_ld16_sync(d + c, v);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mine[(c / 4 + k) * kRows] = make_float4(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]),
                                                                __uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3]));
                }
                __threadfence();
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (threadIdx.x == 64) {
                    // the columns for which this CTA is the last of the tile's; the pairs begin at different
                    // ones, so that those which end together share the additions
                    int* count = reinterpret_cast<int*>(ws + P.off_count) + (2 * it.j + rank) * kJoins;
                    int seen[kJoins], last = 0;
                    const int at = (me - w0) * joins / (w1 - w0 + 1);
#pragma unroll
                    for (int b = 0; b < kJoins; ++b)
                        if (b < joins) seen[b] = atomicAdd(count + (at + b) % joins, 1);
#pragma unroll
                    for (int b = 0; b < kJoins; ++b)
                        if (b < joins && seen[b] == w1 - w0) last |= 1 << (at + b) % joins;
                    bars->last = last;
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                const int last = bars->last;
                joined |= last << joined_at(it.j);
                if (last) __threadfence();
                // add the partials in order, this CTA's own from the accumulator; the others' are requested three
                // pairs at a time, one round trip each
                for (int c = 0; c < toks; c += kJoinCols) {
                    if (!(last >> c / kJoinCols & 1)) continue;
                    uint32_t own[32];
                    tmem_ld32_sync(d + c, own);
                    float v[32] = {};
                    bool mine_in = false;
                    auto add_own = [&] {
                        mine_in = true;
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[k] += __uint_as_float(own[k]);
                    };
                    for (int o = 0; o < w1 - w0; o += 3) {
                        float4 y[3][8];
#pragma unroll
                        for (int i = 0; i < 3; ++i)
                            if (o + i < w1 - w0) {
                                const int wa = w0 + o + i + (w0 + o + i >= me);
                                const float4* src = part(wa) + c / 4 * kRows;
#pragma unroll
                                for (int k = 0; k < 8; ++k)
                                    if (k < 4 || c + 16 < toks) y[i][k] = __ldcg(src + k * kRows);
                            }
#pragma unroll
                        for (int i = 0; i < 3; ++i)
                            if (o + i < w1 - w0) {
                                if (!mine_in && w0 + o + i >= me) add_own();
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    v[4 * k] += y[i][k].x;
                                    v[4 * k + 1] += y[i][k].y;
                                    v[4 * k + 2] += y[i][k].z;
                                    v[4 * k + 3] += y[i][k].w;
                                }
                            }
                    }
                    if (!mine_in) add_own();
                    store16(c, v);
                    if (c + 16 < toks) store16(c + 16, v + 16);
                }
            }
            release();
        }
        if (__any_sync(0xffffffffu, broken)) {
            // once more over what this CTA stored, for the outputs that are to be computed again
            Walk again(P);
            while (again.next(P, &it)) {
                const int blk = it.tile % P.nb, toks = min(P.tb, P.M - blk * P.tb);
                const uint32_t mine = it.j >= 0 ? joined >> joined_at(it.j) : ~0u;
                if (reinterpret_cast<const int2*>(ws + P.off_meta)[static_cast<size_t>(blk) * (P.slots + 1)].x == 0) continue;
                for (int c = it.lo; c < min(it.lo + it.cols, toks); c += 16)
                    if (mine >> c / kJoinCols & 1)
                        own_columns<T>(A, P, ws, blk, c, it.tile / P.nb * 2 * kRows + static_cast<int>(rank) * kRows + 32 * (warp & 3), toks, bars->perm);
            }
        }
    }
    // ---- teardown
    __syncthreads();
    if (threadIdx.x == 0 && *err != 0) {
        // after a failure, loads or arrivals may still be in flight towards either CTA
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 20000ull) {
        }
    }
    tc_fence_before();
    cluster_sync();   // no CTA leaves (or frees tensor memory) while the pair may still address it
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tbase, 512);
}

// ------------------------------------------------------------------------------------- a few tokens

// 16 bytes that are used once (X, which every row of W meets, keeps its place in L1)
__device__ __forceinline__ uint4 load_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Up to kFewTokens tokens: a warp takes two weight rows at a time, 16 bytes of each a lane and step, and
// adds the tokens' adapters (U from the shrink kernel) before its lanes' sums meet. All that counts is
// the stream of W: 32 warps an SM keep 64 KB of it in flight (16 warps with four steps each: 20.3 us for
// one token onto 8192 rows of 5120, 32 with two: 16.8; onto 65536 rows of 7168 139 us, 6.8 TB/s).
template <typename T, int kM>
__global__ void __launch_bounds__(32 * kGemvWarps, kGemvBlocks) lora_gemv_kernel(const LoraArgs A, const Plan P, unsigned char* ws) {
    const int lane = threadIdx.x & 31, warps = gridDim.x * kGemvWarps;
    const T* x = static_cast<const T*>(A.x);
    const float* u[kM];    // the token's row of U in fp32, or none
    long long b_row[kM];   // its adapter's first row of B
    bool ready = false;
    for (int pair = blockIdx.x * kGemvWarps + threadIdx.x / 32; pair * 2 < P.N; pair += warps) {
        const int n0 = 2 * pair, n1 = min(n0 + 1, P.N - 1);
        const T* w0 = static_cast<const T*>(A.w) + static_cast<long long>(n0) * P.K;
        const T* w1 = static_cast<const T*>(A.w) + static_cast<long long>(n1) * P.K;
        float acc[2][kM] = {};
        auto add = [&](const uint4& v0, const uint4& v1, const uint4& xs, int m) {
            float f0[8], f1[8], y[8];
            to_float8<T>(v0, f0);
            to_float8<T>(v1, f1);
            to_float8<T>(xs, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[0][m] = fmaf(f0[i], y[i], acc[0][m]);
                acc[1][m] = fmaf(f1[i], y[i], acc[1][m]);
            }
        };
        for (int k0 = 8 * lane; k0 < P.K; k0 += 256 * kGemvSteps) {
            uint4 v[2][kGemvSteps];
#pragma unroll
            for (int j = 0; j < kGemvSteps; ++j)
                if (k0 + 256 * j < P.K) {
                    v[0][j] = load_once(w0 + k0 + 256 * j);
                    v[1][j] = load_once(w1 + k0 + 256 * j);
                }
#pragma unroll
            for (int j = 0; j < kGemvSteps; ++j)
                if (k0 + 256 * j < P.K)
#pragma unroll
                    for (int m = 0; m < kM; ++m)
                        if (m < P.M)
                            add(v[0][j], v[1][j], __ldg(reinterpret_cast<const uint4*>(x + m * A.x_stride + k0 + 256 * j)), m);
        }
        if (!ready) {
            ready = true;
            pdl_wait();
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                const int id = m < P.M ? A.ids[m] : -1;
                const bool one = id >= 0 && id < P.adapters;
                u[m] = one ? u32_row(P, ws, 0, m) : nullptr;
                b_row[m] = one ? static_cast<long long>(id) * P.N : 0;
            }
        }
#pragma unroll
        for (int m = 0; m < kM; ++m)
            if (u[m])
                for (int k = 8 * lane; k < P.r; k += 256) {
                    const T* b = static_cast<const T*>(A.b);
                    const float4 u0 = __ldcg(reinterpret_cast<const float4*>(u[m] + k)), u1 = __ldcg(reinterpret_cast<const float4*>(u[m] + k + 4));
                    const float y[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
                    float f0[8], f1[8];
                    to_float8<T>(load_once(b + (b_row[m] + n0) * P.r + k), f0);
                    to_float8<T>(load_once(b + (b_row[m] + n1) * P.r + k), f1);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        acc[0][m] = fmaf(f0[i], y[i], acc[0][m]);
                        acc[1][m] = fmaf(f1[i], y[i], acc[1][m]);
                    }
                }
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float y = acc[i][m];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
                if (lane == 2 * m + i && m < P.M && n0 + i < P.N)
                    static_cast<T*>(A.y)[static_cast<long long>(m) * P.N + n0 + i] = ElemTraits<T>::from_f(y);
            }
    }
    if (!ready) pdl_wait();
}

template <typename T>
cudaError_t launch(const LoraArgs& A, unsigned char* ws, int sms, cudaStream_t s) {
    const Plan P = make_plan(A.M, A.N, A.K, A.adapters, A.rank, sms);
    const bool few = A.M <= kFewTokens;
    Maps maps;
    const uint64_t K = static_cast<uint64_t>(A.K), N = static_cast<uint64_t>(A.N), r = static_cast<uint64_t>(A.rank);
    const uint64_t wd[2] = {K, N}, ws1[1] = {K * 2};
    const uint64_t xd[2] = {K, static_cast<uint64_t>(A.M)}, xs[1] = {(P.sorted ? K : static_cast<uint64_t>(A.x_stride)) * 2};
    const uint64_t bd[3] = {r, N, static_cast<uint64_t>(A.adapters)}, bs[2] = {r * 2, r * N * 2};
    const uint64_t kw = static_cast<uint64_t>(P.kw);
    const uint64_t ud[2] = {kw, static_cast<uint64_t>(P.nb) * P.slots * P.rchunks * P.tb}, us[1] = {kw * 2};
    const uint32_t half = static_cast<uint32_t>(P.tb) / 2;
    const uint32_t sb[2] = {kChunk, static_cast<uint32_t>(P.slice) / 2};
    const uint32_t wb[2] = {kChunk, kRows}, xb[2] = {kChunk, half}, bb[3] = {static_cast<uint32_t>(P.kw), kRows, 1},
                   ub[2] = {static_cast<uint32_t>(P.kw), kColStep / 2};
    const CUtensorMapSwizzle rswz = P.kw == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : P.kw == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                                                         : CU_TENSOR_MAP_SWIZZLE_32B;
    if (!few && (!encode_tmap_16b(&maps.w, A.w, 2, wd, ws1, wb, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tmap_16b(&maps.x, P.sorted ? ws + P.off_x : A.x, 2, xd, xs, xb, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tmap_16b(&maps.xs, P.sorted ? ws + P.off_x : A.x, 2, xd, xs, sb, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tmap_16b(&maps.b, A.b, 3, bd, bs, bb, rswz) ||
        !encode_tmap_16b(&maps.u, ws + P.off_u, 2, ud, us, ub, rswz)))
        return cudaErrorInvalidValue;
    const int smem = P.stages * P.stage_bytes + static_cast<int>(sizeof(Bars)) + 1024;
    cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(lora_gemm_kernel<T>),
                                        kSmemCap + static_cast<int>(sizeof(Bars)) + 1024);
    if (e != cudaSuccess) return e;
    const int steps = shrink_steps(P.rsteps);
    const auto shrink = steps == 4 ? lora_shrink_kernel<T, 4> : steps == 2 ? lora_shrink_kernel<T, 2> : lora_shrink_kernel<T, 1>;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = P.ksplit;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(P.clusters * P.ksplit);
    cfg.blockDim = dim3(32 * kShrinkWarps);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if ((e = cudaLaunchKernelEx(&cfg, shrink, A, P, ws)) != cudaSuccess) return e;
    // the GEMM is let in as soon as all CTAs of the shrink kernel run
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    if (few) {
        const int blocks = ceil_div(ceil_div(P.N, 2), kGemvWarps);
        cfg.gridDim = dim3(blocks < kGemvBlocks * sms ? blocks : kGemvBlocks * sms);
        cfg.blockDim = dim3(32 * kGemvWarps);
        e = A.M == 1 ? cudaLaunchKernelEx(&cfg, lora_gemv_kernel<T, 1>, A, P, ws)
                     : cudaLaunchKernelEx(&cfg, lora_gemv_kernel<T, kFewTokens>, A, P, ws);
        count_launches(2);
        return e != cudaSuccess ? e : cudaGetLastError();
    }
    cfg.gridDim = dim3(2 * P.pairs);
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = smem;
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
