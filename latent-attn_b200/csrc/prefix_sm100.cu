// Shared-prefix decode attention on the tensor cores (tcgen05 + TMEM + TMA), d_c = 512, d_R = 64.
//
// Three kernels, chained by programmatic dependent launch:
//   1. prefix_plan_kernel (one block) cuts the query rows into groups of up to 128 and counts their
//      64-position tiles, from the lengths on the device.
//   2. prefix_attend_kernel streams the tiles: one worker is a pair of CTAs, the tiles of all groups
//      are laid end to end and cut evenly over the workers, and a worker writes one partial record
//      (m, l, o) per group that it touches, at index group + worker (unique: walking the tiles in
//      order, every step to the next (group, worker) piece advances one of the two).
//   3. prefix_merge_kernel merges each output row's records by their maxima and sums, once the row's own
//      workers have written them.
// Rounding: P is rounded to the cache's type for its MMA, and the row sums add the rounded values, so
// that the weights of a row still add up to one; a record's o is stored in fp16 after an exact scaling
// of each 64 columns by a power of two (2^-11 relative to their largest, at half of fp32's bytes); all sums, maxima and accumulators are fp32; the result is rounded once.
// A group is the M = 128 tile of the MMAs. When 128 divides H it is 128 heads of one request, whose
// positions are its prefix followed by its own rows. Otherwise the (request, head) rows of a prefix
// group are packed across requests, so that one pass over the prefix serves 128 / H requests, and
// each request's own rows are a group of their own.
//
// The pair splits both products evenly and reads every cache byte into shared memory once: CTA r
// holds columns [256 r, 256 r + 256) of the latent and [32 r, 32 r + 32) of the rope key; it computes
// the partial scores over them, and the output columns [256 r, + 256). TMEM per CTA: O 256 columns |
// two score buffers of 64 | Q latent 128 (two elements a column). (The alternatives: a whole score in
// each CTA costs 1.53 times the MMAs; splitting the rows instead needs every value column twice in
// shared memory, and those MMAs with both operands there ran at 1319 TFLOP/s alone, 868 with their
// loads.) The partial scores cross through distributed shared memory, 24 bits each: a row of a tile as
// integers of 23 bits under one power of two, 2^-22 to 2^-23 of the row's largest partial, where the sums
// of products themselves are good to about 2^-23 of it. A row whose partials reach 2^14 (in log2 units; a
// mask's lowest value, infinities and NaN among them) crosses as floats of 16 significant bits, so that one
// such partial does not take the others' bits. Both CTAs add the same two values, so their softmax is the
// same bit for bit. (32 bits: 20 percent more time with the three loading stages that leave room for them,
// 14 with two exchange slots and P in a place of its own; 16 as fp16: 12 percent less, but then a weight is
// off by 2^-11 of its score.)
//
// Warps (128 + 128 kSets threads): warp 0 loads, warp 1 issues the scores' MMAs and warp 2 the value
// products' (two warps that sleep on their own barriers: one that polls both sees either 0.4 us later),
// warp 3 rests; softmax set i takes the tiles j with j % kSets == i, thread = query row. A tile's way
// through the softmax (read S, exchange, maximum, exponentials, write P) is about 3.5 us of latency with
// little issue time, so kSets tiles are under way at once, each in a slot of its own: the peer's partial
// scores arrive in it, row by row in the layout of an MMA operand, and each thread replaces its row by
// its row of P, from which the value product reads. The MMA that has read it tells the peer that the
// slot is free.
// Bound by that chain and the MMAs: a tile takes 1.30 us (0.78 at the measured tensor rate), a batch 16 us
// beside its tiles (plan 4, first loads 3, last softmax and record 4, merge 3, launches), a group of its
// own about 3. 64 requests of 128 heads
// over a prefix of 8192: 178 us, 843 TFLOP/s; 32 of 16 heads over one of 131072: 171 us, 853 TFLOP/s.
// A parity wait may only start once the phase before the awaited one is known to be complete (it would
// pass at once otherwise), so a barrier that a set waits on for its own tiles belongs to that set.
#include <cfloat>

#include "mla_internal.cuh"
#include "ops.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

namespace mla {
using namespace sm100;

namespace {

constexpr int kTile = 64;                            // positions per tile
constexpr int kStages = 4;
constexpr int kChunkBytes = kTile * 128;             // 64 rows x 64 latent columns, 128-byte swizzle
constexpr int kRopeBoxBytes = kTile * 16;            // 64 rows x 8 rope columns, no swizzle
constexpr int kRopeBytes = 4 * kRopeBoxBytes;
constexpr int kStageBytes = kRopeBytes + 4 * kChunkBytes;
constexpr int kXBytes = 128 * 192;                   // a slot: 128 rows x 64 partial scores of 24 bits, then P in 16
constexpr int kQRopeBoxBytes = 128 * 16;
constexpr int kQRopeBytes = 4 * kQRopeBoxBytes;
constexpr int kXUnit = 128 * 16;                     // 16-byte unit c of row t is at c * kXUnit + t * 16: a warp's stores
                                                     // fill whole sectors on their way to the peer
constexpr int kMSlots = 4;
constexpr int kSets = 3;
constexpr int kSlots = 3;                            // exchange and P slots, tile j in slot j % kSlots
constexpr int kSums = 2 * kSlots;                    // row sums handed between the sets, tile j's in j % kSums
constexpr int kGroupCost = 4;                        // a group's fixed cost, in tiles, for the split (a batch of
                                                     // questions about a document of 131072: 2: 178 us, 4: 171, 6: 176)
constexpr int kThreads = 128 + 128 * kSets;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 0, kColS = 256, kColQ = 384;
constexpr int kMl = 12;
constexpr float kRescale = 8.0f;                     // log2 units
constexpr float kLowest = -FLT_MAX;                  // reference of rows whose scores are all -inf
constexpr float kMagic = 12582912.0f;                // 1.5 * 2^23: x + kMagic holds the integer nearest to x in its low 23 bits
constexpr uint32_t kWideExp = 127 + 14;              // rows whose partials reach 2^14 cross as floats of 24 bits

enum : int { kWaitLoad = 1, kWaitMma = 3, kWaitS = 7, kWaitX = 8, kWaitPV = 9, kWaitTeardown = 10, kWaitDrain = 11,
             kWaitRef = 12, kWaitCredit = 13, kWaitEpi = 14, kAlignment = 15 };

// A group of query rows with something to attend to.
struct __align__(16) Group {
    int q_row0, rows;         // flattened (request, head) rows
    int pid, sid;             // prefix group and request whose rows it attends to (-1: none)
    int plen, slen;
    int tile0, ptiles;        // first tile, tiles of the prefix
    int tile1, pad[3];        // end of its tiles
};
// What a worker starts with.
struct __align__(16) Start {
    int tb, te;               // its tiles
    int g, pad;               // the first one's group, and that group
    Group d;
};
// Where a row finds its records: group + worker for the workers w0 .. w1 (none: w0 > w1).
struct __align__(16) Pieces {
    int g, w0, w1, pad;
};
struct Work {                 // workspace
    int* status;
    int* unsorted;            // group_starts decreases somewhere: no group is built, every output is NaN
    Group* group;             // groups with tiles, in order
    Start* start;             // per worker
    Pieces* pieces;           // per group, also those without tiles: single requests' first, then the prefixes'
    int2* request;            // per request: its prefix's first group among `pieces` (or -1) and first row
    int* gbase;               // per prefix group: its first row group (num_groups + 1)
    int* bad;                 // per group with tiles: it met a row outside the cache
    int* done;                // per worker: its CTAs that have begun, and those whose records are written
    float* rec_ml;            // per record row kMl floats: m, l, -, -, and 2^-f of each 64 columns of o
    uint16_t* rec_o;          // o 2^f in fp16
    float2* rowsum;           // per CTA: [kSums][128] row sums and references handed between its sets
    int W;                    // workers
    int own;                  // groups of single requests (B * ceil(H / 128))
    int fold;                 // 1: prefix and own rows in one group (128 divides H)
};

__device__ __forceinline__ int code(int site) { return kStatusTimeout | (site << 8); }
__device__ __forceinline__ bool warp_ok(bool ok) { return __all_sync(0xffffffffu, ok); }
__device__ __forceinline__ int clampi(int v, int hi) { return v < 0 ? 0 : (v > hi ? hi : v); }

// Prefix group of request b, or -1: the last one that starts at or before b, if it holds b.
__device__ __forceinline__ int prefix_of(const int* starts, int P, int b) {
    int lo = 0, hi = P;
    while (lo + 1 < hi) {
        const int mid = (lo + hi) / 2;
        if (starts[mid] <= b) lo = mid; else hi = mid;
    }
    return starts[lo] <= b && b < starts[lo + 1] ? lo : -1;
}

// ------------------------------------------------------------------------------------- plan

constexpr int kPlanThreads = 1024;  // most; 256 where they cover the groups (fewer warps meet at the barriers)
constexpr int kPlanGroups = 256;    // groups with tiles that are kept in shared memory
constexpr int kPlanCache = 4096;   // groups (and prefix groups) whose sums are kept in shared memory
constexpr int kMaxWorkers = 128;

// Exclusive sums over the block's threads of v (two 32-bit counts in one); *carry is advanced by their total.
__device__ long long block_scan(long long v, long long* sh, long long* carry) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    long long before = 0, total = 0;
    {
        long long s = lane < blockDim.x / 32 ? sh[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        total = __shfl_sync(0xffffffffu, s, 31);
        before = __shfl_sync(0xffffffffu, s, warp > 0 ? warp - 1 : 0);
    }
    const long long at = *carry + x - v + (warp ? before : 0);
    __syncthreads();
    if (threadIdx.x == 0) *carry += total;
    __syncthreads();
    return at;
}

// One block. Latency is all that counts here: one round of loads for everything, the searches in shared
// memory (in global memory beyond kPlanCache).
__global__ void __launch_bounds__(kPlanThreads) prefix_plan_kernel(const __grid_constant__ PrefixArgs A, const Work wk) {
    __shared__ long long sh[32], carry;
    __shared__ int sh_starts[kPlanCache / 4 + 1], sh_plens[kPlanCache / 4];
    __shared__ int sh_base[kPlanCache / 4 + 1];        // gbase
    __shared__ int sh_unit[kPlanCache + 1];            // per group with tiles: tiles and fixed costs before it
    __shared__ Group sh_group[kPlanGroups];
    __shared__ int sh_cut[kMaxWorkers + 1];            // where each share begins
    __shared__ int sh_tile[kMaxWorkers + 1];           // per worker with tiles: its first one
    __shared__ unsigned sh_has[kMaxWorkers / 32];
    pdl_launch_dependents();
    const int hb = ceil_div(A.H, 128), tid = threadIdx.x, threads = blockDim.x;
    const int len0 = tid < wk.own ? A.lens[tid / hb] : 0;   // this thread's first own group
    const bool base_sh = A.P <= kPlanCache / 4;
    int falls = 0;
    for (int p = tid; p < A.P; p += threads) {
        const int s0 = A.starts[p], s1 = A.starts[p + 1];
        falls |= s0 > s1;
        if (base_sh) {
            sh_starts[p] = s0;
            if (p + 1 == A.P) sh_starts[A.P] = s1;
            sh_plens[p] = A.plens[p];
        }
    }
    const int* starts = base_sh ? sh_starts : A.starts;
    const int* plens = base_sh ? sh_plens : A.plens;
    if (tid == 0) {
        carry = 0;
        *wk.status = 0;
    }
    if (tid < wk.W) wk.done[tid] = 0;
    // the tables hold the groups of disjoint ranges of requests; ranges that fall back could be any number
    const bool sorted = !__syncthreads_or(falls);
    if (tid == 0) *wk.unsorted = !sorted;
    int extra = 0;   // row groups of the prefixes
    if (!wk.fold && sorted) {
        for (int p0 = 0; p0 < A.P; p0 += threads) {
            const int p = p0 + tid;
            int n = 0;
            if (p < A.P) {
                const int s0 = max(starts[p], 0), s1 = min(starts[p + 1], A.B);
                n = s1 > s0 ? static_cast<int>((static_cast<long long>(s1 - s0) * A.H + 127) / 128) : 0;
            }
            const int at = static_cast<int>(block_scan(n, sh, &carry));
            if (p < A.P) {
                if (base_sh) sh_base[p] = at;
                else wk.gbase[p] = at;
            }
        }
        extra = static_cast<int>(carry);
        __syncthreads();
        if (tid == 0) carry = 0;
        __syncthreads();
    }
    const int* gbase = base_sh ? sh_base : wk.gbase;
    // groups: tiles, then (compacted) the table
    const int G = sorted ? wk.own + extra : 0;
    int mine = -1, mine0 = 0, mine1 = 0;   // this thread's last group: its place in the table, its tiles
    for (int g0 = 0; g0 < G; g0 += threads) {
        const int g = g0 + tid;
        Group d = {};
        int tiles = 0;
        if (g < wk.own) {
            const int b = g / hb, k = g % hb;
            const int p = prefix_of(starts, A.P, b);
            d.q_row0 = b * A.H + 128 * k;
            d.rows = min(128, A.H - 128 * k);
            d.pid = wk.fold ? p : -1;
            d.sid = b;
            d.plen = d.pid >= 0 ? clampi(plens[d.pid], A.max_plen) : 0;
            d.slen = clampi(g0 == 0 ? len0 : A.lens[b], A.max_len);
            if (!wk.fold && k == 0)
                wk.request[b] = p < 0 ? make_int2(-1, 0) : make_int2(wk.own + gbase[p], max(starts[p], 0) * A.H);
        } else if (g < G) {
            const int e = g - wk.own;
            int lo = 0, hi = A.P;   // last prefix group that starts at or before e
            while (lo + 1 < hi) {
                const int mid = (lo + hi) / 2;
                if (gbase[mid] <= e) lo = mid; else hi = mid;
            }
            const int s0 = max(starts[lo], 0), s1 = min(starts[lo + 1], A.B);
            const int at = (e - gbase[lo]) * 128;
            d.q_row0 = s0 * A.H + at;
            d.rows = min(128, (s1 - s0) * A.H - at);
            d.pid = lo;
            d.sid = -1;
            d.plen = clampi(plens[lo], A.max_plen);
        }
        if (g < G) {
            d.ptiles = ceil_div(d.plen, kTile);
            tiles = d.ptiles + ceil_div(d.slen, kTile);
        }
        const long long at = block_scan(static_cast<long long>(tiles > 0) << 32 | tiles, sh, &carry);
        const int c = static_cast<int>(at >> 32);   // groups with tiles before this one
        d.tile0 = static_cast<int>(at);
        d.tile1 = d.tile0 + tiles;
        mine = tiles > 0 ? c : -1;
        mine0 = d.tile0;
        mine1 = d.tile1;
        if (g < G && G > threads) wk.pieces[g] = {mine, mine0, mine1, 0};   // until the workers are known
        if (tiles > 0) {
            wk.group[c] = d;
            if (c < kPlanGroups) sh_group[c] = d;
            wk.bad[c] = 0;
            if (c < kPlanCache) sh_unit[c] = d.tile0 + c * kGroupCost;
        }
    }
    const int T = static_cast<int>(carry), C = static_cast<int>(carry >> 32);
    __syncthreads();   // the table is complete (this block's writes are visible to it)
    // Worker w begins at w / W of all tiles and fixed costs. A group's cost lies before its tiles; a
    // share that begins there begins with the group. Shares that hold no tile are left out.
    auto unit = [&](int c) { return c < kPlanCache ? sh_unit[c] : wk.group[c].tile0 + c * kGroupCost; };
    int first = 0;   // the group that this thread's share begins with
    if (tid <= wk.W) {
        const long long u = static_cast<long long>(T + C * kGroupCost) * tid / wk.W;
        int lo = 0, hi = C;   // last group whose cost and tiles begin at or before u
        while (lo + 1 < hi) {
            const int mid = (lo + hi) / 2;
            if (unit(mid) <= u) lo = mid; else hi = mid;
        }
        const int tile0 = C > 0 ? unit(lo) - lo * kGroupCost : 0;
        const int tile1 = lo + 1 < C ? unit(lo + 1) - (lo + 1) * kGroupCost : T;
        const long long x = u - static_cast<long long>(lo + 1) * kGroupCost;
        const int cut = tid == wk.W ? T : static_cast<int>(x < tile0 ? tile0 : (x > tile1 ? tile1 : x));
        sh_cut[tid] = cut;
        first = cut == tile1 ? lo + 1 : lo;
    }
    __syncthreads();
    const bool has = tid < wk.W && sh_cut[tid] < sh_cut[tid + 1];
    if (tid < kMaxWorkers) {
        const unsigned mask = __ballot_sync(0xffffffffu, has);
        if ((tid & 31) == 0) sh_has[tid / 32] = mask;
    }
    __syncthreads();
    int workers = 0, at = 0;
#pragma unroll
    for (int i = 0; i < kMaxWorkers / 32; ++i) {
        if (i < tid / 32) at += __popc(sh_has[i]);
        workers += __popc(sh_has[i]);
    }
    if (has) {
        at += __popc(sh_has[tid / 32] & ((1u << (tid & 31)) - 1));
        sh_tile[at] = sh_cut[tid];
        Start st;
        st.tb = sh_cut[tid];
        st.te = sh_cut[tid + 1];
        st.g = first;
        st.pad = 0;
        st.d = first < kPlanGroups ? sh_group[first] : wk.group[first];
        wk.start[at] = st;
    }
    if (tid >= workers && tid < wk.W) wk.start[tid].tb = wk.start[tid].te = 0;
    __syncthreads();
    // the workers of each group
    for (int g = tid; g < G; g += threads) {
        if (G > threads) {
            const Pieces p = wk.pieces[g];
            mine = p.g;
            mine0 = p.w0;
            mine1 = p.w1;
        }
        auto worker = [&](int t) {   // the last one that begins at or before tile t
            int lo = 0, hi = workers;
            while (lo + 1 < hi) {
                const int mid = (lo + hi) / 2;
                if (sh_tile[mid] <= t) lo = mid; else hi = mid;
            }
            return lo;
        };
        wk.pieces[g] = {mine, mine >= 0 ? worker(mine0) : 0, mine >= 0 ? worker(mine1 - 1) : -1, 0};
    }
}

// ------------------------------------------------------------------------------------- attend

struct __align__(8) Barriers {
    uint64_t kv_full[kStages], kv_empty[kStages];
    uint64_t s_full[kSets];           // per set: the score of its next tile is done
    uint64_t s_free[2];               // per score buffer (tile parity): it has been read
    uint64_t x_full[kSlots];          // the peer's partial scores have arrived in the slot
    uint64_t p_full[kSlots];          // the slot holds P
    uint64_t pv_done[kSlots];         // the value product has read it
    uint64_t x_empty[kSlots];         // and so it has in the peer, whose slot may be written again
    uint64_t mref[kMSlots];           // m_pub slot j % kMSlots holds tile j's reference
    uint64_t lpub[kSums];           // rowsum slot j % kSums holds tile j's set's sums (near a segment's end)
    uint64_t q_first, q_ready;        // the first group's Q is in place; a later one's
    uint64_t o_free, drain[2], done;
    uint32_t tmem;
};

constexpr size_t kSmemBytes = static_cast<size_t>(kStages) * kStageBytes + static_cast<size_t>(kSlots) * kXBytes +
                              kQRopeBytes + kMSlots * 128 * sizeof(float) + sizeof(Barriers) + kSlots * 128;
static_assert(kSmemBytes <= 232448, "shared memory budget");

// Walks a worker's tiles; every role walks an identical copy. A segment is the worker's run of tiles
// of one group.
struct Tiles {
    int t, t_end, g, seg0;
    Group d;
    __device__ void init(const Start& st) {
        t = seg0 = st.tb;
        t_end = st.te;
        g = st.g;
        d = st.d;
    }
    __device__ bool valid() const { return t < t_end; }
    __device__ bool own() const { return t - d.tile0 >= d.ptiles; }
    __device__ int pos0() const { return (t - d.tile0 - (own() ? d.ptiles : 0)) * kTile; }
    __device__ int np() const { return min(kTile, (own() ? d.slen : d.plen) - pos0()); }
    __device__ int seg_tile() const { return t - seg0; }
    __device__ bool seg_first() const { return t == seg0; }
    __device__ int seg_end() const { return min(t_end, d.tile1); }
    __device__ bool seg_last() const { return t + 1 == seg_end(); }
    __device__ void next(const Work& wk) {
        ++t;
        if (t == d.tile1 && t < t_end) {
            d = wk.group[++g];
            seg0 = t;
        }
    }
    __device__ void skip(const Work& wk, int n) {
        for (; n > 0 && valid(); --n) next(wk);
    }
};

template <typename T> struct Fmt;
template <> struct Fmt<__half> { static constexpr uint32_t v = 0; };
template <> struct Fmt<__nv_bfloat16> { static constexpr uint32_t v = 1; };

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// volatile: keeps a run of them together
__device__ __forceinline__ float ex2_ordered(float x) {
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ uint32_t pair_of(float a, float b);
template <> __device__ __forceinline__ uint32_t pair_of<__half>(float a, float b) { return half2_of(a, b); }
template <> __device__ __forceinline__ uint32_t pair_of<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float2 floats_of(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
// two fp32 lanes in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
// the largest magnitude of three (NaN if one is)
__device__ __forceinline__ float maxabs3(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Three bytes of each of four words in three, and back (the top byte of each is then kMagic's).
__device__ __forceinline__ void pack24(const float* x, uint32_t* w) {
    const uint32_t a = __float_as_uint(x[0]), b = __float_as_uint(x[1]), c = __float_as_uint(x[2]), d = __float_as_uint(x[3]);
    w[0] = __byte_perm(a, b, 0x4210);
    w[1] = __byte_perm(b, c, 0x5421);
    w[2] = __byte_perm(c, d, 0x6542);
}
__device__ __forceinline__ void unpack24(const uint32_t* w, float* x) {
    constexpr uint32_t k = 0x4B000000u;
    x[0] = __uint_as_float(__byte_perm(w[0], k, 0x7210));
    x[1] = __uint_as_float((__byte_perm(w[0], w[1], 0x5543) & 0x00FFFFFFu) | k);
    x[2] = __uint_as_float((__byte_perm(w[1], w[2], 0x4432) & 0x00FFFFFFu) | k);
    x[3] = __uint_as_float(__byte_perm(w[2], k, 0x7321));
}
// A float rounded to 24 bits (16 significant ones), and back.
__device__ __forceinline__ float to_wide24(float x) {
    return __uint_as_float(x != x ? 0x7FC000u : (__float_as_uint(x) + 0x80u) >> 8);
}
__device__ __forceinline__ float from_wide24(float w) { return __uint_as_float(__float_as_uint(w) << 8); }
// the largest of three (a NaN only if all are)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 32 bytes a lane, in one request where the address allows it: lanes on different rows cost one tag each
// and request.
__device__ __forceinline__ void load32(const uint4* p, bool aligned, uint4& a, uint4& b) {
    if (aligned) {
        asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                     : "l"(p));
    } else {
        a = __ldg(p);
        b = __ldg(p + 1);
    }
}

// 64 columns of this thread's O row (TMEM) to a record row, times the 2^f that brings them below 2^15
// (1 for zeros, and for infinities and NaN, which go into the record as they are); returns 2^-f.
// Warp-collective.
__device__ __forceinline__ float write_cols(uint32_t tsrc, uint16_t* orow, bool row_ok) {
    uint32_t o[64];
    tmem_ld64_sync(tsrc, o);
    float mx[4] = {};
#pragma unroll
    for (int i = 0; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], fabsf(__uint_as_float(o[i])));
    // exponent field of 2^(14 - floor(log2 top)), kept where both 2^f and 2^-f are normal
    const int e = static_cast<int>(__float_as_uint(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]))) >> 23);
    const int f = e > 0 && e < 255 ? min(max(268 - e, 1), 253) : 127;
    const float scale = __uint_as_float(static_cast<uint32_t>(f) << 23);
    if (row_ok) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = half2_of(__uint_as_float(o[16 * q + 2 * i]) * scale, __uint_as_float(o[16 * q + 2 * i + 1]) * scale);
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(orow + 16 * q),
                         "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                         : "memory");
        }
    }
    return __uint_as_float(static_cast<uint32_t>(254 - f) << 23);
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
prefix_attend_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ CUtensorMap tmap_rope,
                     const __grid_constant__ PrefixArgs A, const __grid_constant__ Work wk) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* stages = smem_raw;   // swizzled tiles want 1024 bytes; there is no room to align it by hand
    unsigned char* xbuf = stages + kStages * kStageBytes;
    unsigned char* qrope = xbuf + kSlots * kXBytes;
    float* m_pub = reinterpret_cast<float*>(qrope + kQRopeBytes);              // [kMSlots][128]
    Barriers* bars = reinterpret_cast<Barriers*>(m_pub + kMSlots * 128);
    unsigned char* xexp = reinterpret_cast<unsigned char*>(bars + 1);          // [kSlots][128] exponents of a slot's rows
    // the row sums that one set hands to another at a segment's end: in global memory, where shared
    // memory has no room, and only for the segment's last tiles
    volatile float2* l_pub = wk.rowsum + static_cast<long long>(blockIdx.x) * kSums * 128;
    const uint32_t rank = cluster_ctarank(), peer = rank ^ 1u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int w = blockIdx.x >> 1;
    volatile int* err = wk.status;

    if (smem_u32(smem_raw) % 1024 != 0) {   // (all CTAs alike)
        pdl_wait();
        if (threadIdx.x == 0) {
            record_timeout(err, code(kAlignment));
            __threadfence();
            atomicAdd(&wk.done[w], 2);
        }
        pdl_launch_dependents();
        return;
    }
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmap);
        tma_prefetch_desc(&tmap_rope);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&bars->kv_full[s]), 1);
            mbar_init(smem_u32(&bars->kv_empty[s]), 1);
        }
        for (int i = 0; i < kSets; ++i) mbar_init(smem_u32(&bars->s_full[i]), 1);
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(smem_u32(&bars->x_full[i]), 1);
            mbar_init(smem_u32(&bars->p_full[i]), 128);
            mbar_init(smem_u32(&bars->pv_done[i]), 1);
            mbar_init(smem_u32(&bars->x_empty[i]), 1);
        }
        for (int b = 0; b < 2; ++b) mbar_init(smem_u32(&bars->s_free[b]), 128);
        for (int i = 0; i < kMSlots; ++i) mbar_init(smem_u32(&bars->mref[i]), 128);
        for (int i = 0; i < kSums; ++i) mbar_init(smem_u32(&bars->lpub[i]), 128);
        mbar_init(smem_u32(&bars->q_first), 128 * kSets);
        mbar_init(smem_u32(&bars->q_ready), 128);
        mbar_init(smem_u32(&bars->o_free), 128);
        mbar_init(smem_u32(&bars->drain[0]), 1);
        mbar_init(smem_u32(&bars->drain[1]), 1);
        mbar_init(smem_u32(&bars->done), 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&bars->tmem), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tbase = bars->tmem;
    pdl_wait();   // the plan
    // passed on to the merge, which does not wait for the plan itself
    if (threadIdx.x == 0) asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(wk.done + w) : "memory");
    // the merge may start: every CTA whose records it awaits runs
    pdl_launch_dependents();
    // identical in both CTAs of the pair; a pair without tiles goes straight to the teardown
    const Start start = wk.start[w];
    const int n = start.te - start.tb;
    const uint32_t stages_u32 = smem_u32(stages), xbuf_u32 = smem_u32(xbuf), qrope_u32 = smem_u32(qrope), xexp_u32 = smem_u32(xexp);

    if (warp < 4) {
        if (n > 0 && warp == 0 && lane == 0) {
            // ------------------------------------------------------------ loads
            Tiles it;
            it.init(start);
            int issued = 0;
            for (int i = 0; it.valid(); ++i, it.next(wk)) {
                const int st = i % kStages;
                const int pos = it.pos0(), np = it.np();
                long long row;
                if (A.page_rows) {
                    const int pg = it.own() ? A.table[static_cast<long long>(it.d.sid) * A.max_pages + pos / A.page_rows]
                                            : A.ptable[static_cast<long long>(it.d.pid) * A.max_ppages + pos / A.page_rows];
                    row = pg < 0 ? -1 : static_cast<long long>(pg) * A.page_rows + pos % A.page_rows;
                } else {
                    row = (it.own() ? A.offs[it.d.sid] : A.poffs[it.d.pid]) + pos;
                }
                if (row < 0 || row + np > A.kv_rows) {
                    wk.bad[it.g] = 1;
                    row = -2 * kTile;   // outside the tensor: reads zeros
                }
                if (i >= kStages && !mbar_wait(smem_u32(&bars->kv_empty[st]), ((i / kStages) - 1) & 1, err, code(kWaitLoad))) break;
                const uint32_t full = smem_u32(&bars->kv_full[st]), dst = stages_u32 + st * kStageBytes;
                mbar_arrive_expect_tx(full, kStageBytes);
                tma_load_3d(dst + kRopeBytes, &tmap, full, 0, static_cast<int>(row), 4 * static_cast<int>(rank));
                tma_load_3d(dst, &tmap_rope, full, 0, static_cast<int>(row), 4 * static_cast<int>(rank));
                issued = i + 1;
            }
            // the last loads land before shared memory is released
            for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
                mbar_wait(smem_u32(&bars->kv_full[i % kStages]), (i / kStages) & 1, err, code(kWaitLoad), 100000000ull);
        } else if (n > 0 && warp == 1) {
            // ------------------------------------------------------------ scores
            // The whole warp walks the tiles and waits, one elected lane issues. Score i needs its
            // stage, its buffer read out, and at a segment's start the group's Q.
            constexpr uint32_t idesc = idesc_f16(128, kTile, Fmt<T>::v, false, false);
            const uint32_t tQ = tbase + kColQ;
            const uint64_t dqr = smem_desc_noswz(qrope_u32, kQRopeBoxBytes, 128);
            Tiles it;
            it.init(start);
            int seg = 0;
            bool ok = true;
            for (int i = 0; it.valid(); ++i, it.next(wk)) {
                ok = mbar_wait(smem_u32(&bars->kv_full[i % kStages]), (i / kStages) & 1, err, code(kWaitMma)) &&
                     (i < 2 || mbar_wait(smem_u32(&bars->s_free[i & 1]), ((i >> 1) - 1) & 1, err, code(kWaitMma))) &&
                     (!it.seg_first() || (seg == 0 ? mbar_wait(smem_u32(&bars->q_first), 0, err, code(kWaitMma))
                                                   : mbar_wait(smem_u32(&bars->q_ready), (seg - 1) & 1, err, code(kWaitMma))));
                if (!warp_ok(ok)) break;
                if (it.seg_first()) ++seg;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t sa = stages_u32 + (i % kStages) * kStageBytes;
                    const uint64_t dl = smem_desc_sw128(sa + kRopeBytes, 16, 1024);
                    const uint32_t tS = tbase + kColS + 64 * (i & 1);
                    mma_ts(tS, tQ, dl, idesc, 0u);
#pragma unroll
                    for (int k = 1; k < 16; ++k)
                        mma_ts(tS, tQ + 8 * k, dl + static_cast<uint64_t>(((k >> 2) * kChunkBytes + (k & 3) * 32) >> 4), idesc, 1u);
                    const uint64_t dr = smem_desc_noswz(sa, kRopeBoxBytes, 128);
                    mma_ss(tS, dqr, dr, idesc, 1u);
                    mma_ss(tS, dqr + static_cast<uint64_t>((2 * kQRopeBoxBytes) >> 4),
                           dr + static_cast<uint64_t>((2 * kRopeBoxBytes) >> 4), idesc, 1u);
                    mma_commit(smem_u32(&bars->s_full[i % kSets]));
                }
                __syncwarp();
            }
            // every MMA is done before the teardown
            if (elect_one()) mma_commit(smem_u32(&bars->drain[0]));
            __syncwarp();
            mbar_wait(smem_u32(&bars->drain[0]), 0, err, code(kWaitDrain));
        } else if (n > 0 && warp == 2) {
            // ------------------------------------------------------------ value products
            // Product i needs P(i), and at a segment's start the O of the one before read out.
            constexpr uint32_t idesc = idesc_f16(128, 256, Fmt<T>::v, false, true);
            const uint32_t tO = tbase + kColO;
            Tiles it;
            it.init(start);
            int seg = 0;
            bool ok = true;
            for (int i = 0; it.valid(); ++i, it.next(wk)) {
                ok = mbar_wait(smem_u32(&bars->p_full[i % kSlots]), (i / kSlots) & 1, err, code(kWaitMma)) &&
                     (!it.seg_first() || seg == 0 || mbar_wait(smem_u32(&bars->o_free), (seg - 1) & 1, err, code(kWaitMma)));
                if (!warp_ok(ok)) break;
                if (it.seg_first()) ++seg;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t dc = smem_desc_sw128(stages_u32 + (i % kStages) * kStageBytes + kRopeBytes, kChunkBytes, 1024);
                    const uint64_t dp = smem_desc_noswz(xbuf_u32 + (i % kSlots) * kXBytes, kXUnit, 128);
                    mma_ss(tO, dp, dc, idesc, it.seg_first() ? 0u : 1u);
#pragma unroll
                    for (int k = 1; k < kTile / 16; ++k)
                        mma_ss(tO, dp + static_cast<uint64_t>((2 * kXUnit * k) >> 4), dc + static_cast<uint64_t>((2048 * k) >> 4), idesc, 1u);
                    mma_commit(smem_u32(&bars->kv_empty[i % kStages]));
                    mma_commit(smem_u32(&bars->pv_done[i % kSlots]));
                    // the peer awaits this for tile i + kSlots; for the last tiles nobody does, and the peer
                    // may be gone when it arrives
                    if (i + kSlots < n) mma_commit_to(smem_u32(&bars->x_empty[i % kSlots]), static_cast<uint16_t>(1u << peer));
                }
                __syncwarp();
            }
            if (elect_one()) mma_commit(smem_u32(&bars->drain[1]));
            __syncwarp();
            mbar_wait(smem_u32(&bars->drain[1]), 0, err, code(kWaitDrain));
        }
    } else {
        // ---------------------------------------------------------------- softmax sets
        const int sid = (warp - 4) >> 2;
        const int t = (warp & 3) * 32 + lane;             // query row == TMEM lane
        const uint32_t trow = tbase + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
        const float qscale = A.scale * 1.4426950408889634f;
        // Q of a group: this thread's half of its row's CTA columns into TMEM (two elements a column) and
        // two of the four rope boxes
        auto load_q = [&](const Group& d, int c0, int step, uint64_t* ready) {
            const long long row = d.q_row0 + t;
            const uint4* lat = reinterpret_cast<const uint4*>(static_cast<const T*>(A.qa) + row * 512 + 256 * rank);
            const uint4* rope = reinterpret_cast<const uint4*>(static_cast<const T*>(A.qr) + row * 64 + 32 * rank);
            const bool have = t < d.rows, q32 = reinterpret_cast<uintptr_t>(A.qa) % 32 == 0;
#pragma unroll 1
            for (int c = c0; c < 4; c += 2 * step) {   // two blocks of 64 columns a round trip
                uint4 v[2][8], r[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool on = have && c + e * step < 4;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        v[e][2 * k] = v[e][2 * k + 1] = make_uint4(0, 0, 0, 0);
                        if (on) load32(lat + 8 * (c + e * step) + 2 * k, q32, v[e][2 * k], v[e][2 * k + 1]);
                    }
                    r[e] = on ? __ldg(rope + c + e * step) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (c + e * step >= 4) break;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint32_t x[16] = {v[e][4 * q].x, v[e][4 * q].y, v[e][4 * q].z, v[e][4 * q].w,
                                                v[e][4 * q + 1].x, v[e][4 * q + 1].y, v[e][4 * q + 1].z, v[e][4 * q + 1].w,
                                                v[e][4 * q + 2].x, v[e][4 * q + 2].y, v[e][4 * q + 2].z, v[e][4 * q + 2].w,
                                                v[e][4 * q + 3].x, v[e][4 * q + 3].y, v[e][4 * q + 3].z, v[e][4 * q + 3].w};
                        tmem_st16(trow + kColQ + 32 * (c + e * step) + 16 * q, x);
                    }
                    *reinterpret_cast<uint4*>(qrope + (c + e * step) * kQRopeBoxBytes + t * 16) = r[e];
                }
            }
            fence_proxy_async_smem();
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(smem_u32(ready));
        };
        Tiles it;
        bool ok = true;
        if (n > 0) {
            it.init(start);
            load_q(it.d, sid, kSets, &bars->q_first);   // the first group's Q: the sets share it
            it.skip(wk, sid);
        } else {
            it.t = it.t_end = 0;
        }
        float l_self = 0.f, m_l = 0.f;    // sum over this thread's columns of the set's tiles of the segment, and its reference
        for (int j = sid; ok && it.valid(); j += kSets, it.skip(wk, kSets)) {
            const int slot = j % kSlots, np = it.np();
            const uint32_t phase = (j / kSlots) & 1;
            const uint32_t x_row = xbuf_u32 + slot * kXBytes + t * 16;
            const uint32_t x_full = smem_u32(&bars->x_full[slot]);
            bool got = true;
            if (it.seg_first() && j > 0) {
                // A new group: its Q replaces the one that the score of tile j - 1 was the last to read. (This set
                // waits for its score anyway; the one of tile j - 1 would be held up. That barrier is another
                // set's, but its phase before is complete: this set's tile j - kSets came after it.)
                got = mbar_wait(smem_u32(&bars->s_full[(j - 1) % kSets]), ((j - 1) / kSets) & 1, err, code(kWaitS));
                if (!warp_ok(got)) break;
                tc_fence_after();
                load_q(it.d, 0, 1, &bars->q_ready);
            }
            // ---- S_r(j) to registers, release S, put the partial in 24 bits
            got = mbar_wait(smem_u32(&bars->s_full[sid]), (j / kSets) & 1, err, code(kWaitS));
            if (!warp_ok(got)) break;
            if (t == 0) mbar_arrive_expect_tx(x_full, kXBytes + 128);
            tc_fence_after();
            float s[64];
            {
                uint32_t sr[64];
                tmem_ld64_sync(trow + kColS + 64 * (j & 1), sr);
                tc_fence_before();
                mbar_arrive(smem_u32(&bars->s_free[j & 1]));
#pragma unroll
                for (int q = 0; q < 64; ++q) s[q] = __uint_as_float(sr[q]);
            }
            if (np < kTile) {   // what lies past the end must not set the row's exponent
#pragma unroll
                for (int k = 0; k < 64; ++k)
                    if (k >= np) s[k] = 0.f;
            }
            uint32_t ex;
            {
                float mx[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < 64; k += 2) mx[(k / 2) & 3] = maxabs3(mx[(k / 2) & 3], s[k], s[k + 1]);
                // (a little more than the largest, so that it stays below 2^22 after rounding)
                ex = __float_as_uint(maxabs3(maxabs3(mx[0], mx[1], mx[2]), mx[3], 0.f) * qscale * 1.000001f) >> 23;
            }
            // (from 2^64 below 1 on, smaller rows are as good as zero; 255 says that the row crosses as floats)
            const bool wide = ex >= kWideExp || !(qscale < 1e12f), some_wide = __any_sync(0xffffffffu, wide);
            ex = wide ? 255u : max(ex, 64u);
            const float sc = qscale * __uint_as_float((275u - ex) << 23);   // 2^21 to 2^22 for the largest
            if (some_wide) {
#pragma unroll
                for (int k = 0; k < 64; ++k) s[k] = wide ? to_wide24(s[k] * qscale) : fmaf(s[k], sc, kMagic);
            } else {
#pragma unroll
                for (int q = 0; q < 32; ++q) {
                    const float2 v = fma2(make_float2(s[2 * q], s[2 * q + 1]), make_float2(sc, sc), make_float2(kMagic, kMagic));
                    s[2 * q] = v.x;
                    s[2 * q + 1] = v.y;
                }
            }
            uint32_t ex4 = ex << (8 * (lane & 3));   // of four rows
            ex4 |= __shfl_xor_sync(0xffffffffu, ex4, 1);
            ex4 |= __shfl_xor_sync(0xffffffffu, ex4, 2);
            // the peer's value product of tile j - kSlots has read its slot
            got = j < kSlots || mbar_wait_cluster(smem_u32(&bars->x_empty[slot]), phase ^ 1, err, code(kWaitCredit));
            if (!warp_ok(got)) break;
            {
                const uint32_t dst = mapa(x_row, peer), bar = mapa(x_full, peer);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[12];
#pragma unroll
                    for (int q = 0; q < 4; ++q) pack24(s + 16 * c + 4 * q, w + 3 * q);
#pragma unroll
                    for (int q = 0; q < 3; ++q)
                        st_async_v4(dst + (3 * c + q) * kXUnit, w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3], bar);
                }
                if ((lane & 3) == 0) st_async(mapa(xexp_u32 + slot * 128 + t, peer), ex4, bar);
            }
            // this CTA's own values as the peer will see them
            {
                const float inv = __uint_as_float((ex - 21u) << 23), off = -kMagic * inv;
                if (some_wide) {
#pragma unroll
                    for (int k = 0; k < 64; ++k) s[k] = wide ? from_wide24(s[k]) : fmaf(s[k], inv, off);
                } else {
#pragma unroll
                    for (int q = 0; q < 32; ++q) {
                        const float2 v = fma2(make_float2(s[2 * q], s[2 * q + 1]), make_float2(inv, inv), make_float2(off, off));
                        s[2 * q] = v.x;
                        s[2 * q + 1] = v.y;
                    }
                }
            }
            if (np < kTile) {
                // rows past the end: their weights are zero, but zero times what lies there need not be
                unsigned char* sp = stages + (j % kStages) * kStageBytes + kRopeBytes;
                const int units = (kTile - np) * 8;
                for (int v = t; v < 4 * units; v += 128)
                    *reinterpret_cast<uint4*>(sp + (v / units) * kChunkBytes + (np + (v % units) / 8) * 128 + (v % 8) * 16) =
                        make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
            }
            // ---- the whole score, its reference, P into the slot. That the peer's scores are here also says
            // that this CTA's value product of tile j - kSlots is done (the peer waited for it).
            got = mbar_wait_cluster(x_full, phase, err, code(kWaitX));
            if (!warp_ok(got)) break;
            // (stage by stage over all columns: the warp issues in order, so column by column it would wait
            // for every step of every chain)
            {
                uint32_t pe;
                asm volatile("ld.shared.u8 %0, [%1];" : "=r"(pe) : "r"(xexp_u32 + slot * 128 + t));
                const bool pwide = pe == 255u;
                const float inv = __uint_as_float((pe - 21u) << 23), off = -kMagic * inv;
                auto load16 = [&](int c, float* x) {
                    uint32_t w[12];
#pragma unroll
                    for (int q = 0; q < 3; ++q)
                        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(w[4 * q]), "=r"(w[4 * q + 1]), "=r"(w[4 * q + 2]), "=r"(w[4 * q + 3])
                                     : "r"(x_row + (3 * c + q) * kXUnit));
#pragma unroll
                    for (int q = 0; q < 4; ++q) unpack24(w + 3 * q, x + 4 * q);
                };
                if (__any_sync(0xffffffffu, pwide)) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float x[16];
                        load16(c, x);
#pragma unroll
                        for (int q = 0; q < 16; ++q) s[16 * c + q] += pwide ? from_wide24(x[q]) : fmaf(x[q], inv, off);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float x[16];
                        load16(c, x);
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            float* y = s + 16 * c + 2 * q;
                            const float2 v = add2(make_float2(y[0], y[1]), fma2(make_float2(x[2 * q], x[2 * q + 1]),
                                                                              make_float2(inv, inv), make_float2(off, off)));
                            y[0] = v.x;
                            y[1] = v.y;
                        }
                    }
                }
            }
            if (np < kTile) {
#pragma unroll
                for (int k = 0; k < 64; ++k)
                    if (k >= np) s[k] = -INFINITY;
            }
            float mt = max3(s[0], s[1], kLowest);
            {
                float mx[4] = {mt, s[2], s[3], s[4]};
#pragma unroll
                for (int k = 5; k + 1 < 64; k += 2) mx[(k / 2) & 3] = max3(mx[(k / 2) & 3], s[k], s[k + 1]);
                mt = fmaxf(max3(mx[0], mx[1], mx[2]), fmaxf(mx[3], s[64 - 1]));
            }
            // the reference of the tile before, unless this one exceeds it by more than the threshold
            float m = mt, alpha = 1.f;
            bool need = false;
            if (!it.seg_first()) {
                got = mbar_wait(smem_u32(&bars->mref[(j - 1) % kMSlots]), ((j - 1) / kMSlots) & 1, err, code(kWaitRef));
                if (!warp_ok(got)) break;
                const float m_prev = m_pub[((j - 1) % kMSlots) * 128 + t];
                if (mt > m_prev + kRescale) {
                    alpha = ex2(m_prev - mt);
                    need = true;
                } else {
                    m = m_prev;
                }
            }
            m_pub[(j % kMSlots) * 128 + t] = m;
            mbar_arrive(smem_u32(&bars->mref[j % kMSlots]));
            uint32_t pp[32];
            const float2 m2 = make_float2(-m, -m);
#pragma unroll
            for (int q = 0; q < 32; ++q) {
                const float2 d = add2(make_float2(s[2 * q], s[2 * q + 1]), m2);
                s[2 * q] = d.x;
                s[2 * q + 1] = d.y;
            }
#pragma unroll
            for (int q = 0; q < 64; ++q) s[q] = ex2_ordered(s[q]);
#pragma unroll
            for (int q = 0; q < 32; ++q) pp[q] = pair_of<T>(s[2 * q], s[2 * q + 1]);
            if (__any_sync(0xffffffffu, need)) {
                // the reference moved: rescale O (alpha = 1 elsewhere) once PV(j - 1) is done
                got = mbar_wait(smem_u32(&bars->pv_done[(j - 1) % kSlots]), ((j - 1) / kSlots) & 1, err, code(kWaitPV));
                if (!warp_ok(got)) break;
                tc_fence_after();
#pragma unroll 1
                for (int c0 = 0; c0 < 256; c0 += 32) {
                    uint32_t o[32];
                    tmem_ld32_sync(trow + kColO + c0, o);
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                    tmem_st32(trow + kColO + c0, o);
                }
                tmem_st_wait();
                tc_fence_before();
            }
#pragma unroll
            for (int c = 0; c < 8; ++c)
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(x_row + c * kXUnit),
                             "r"(pp[4 * c]), "r"(pp[4 * c + 1]), "r"(pp[4 * c + 2]), "r"(pp[4 * c + 3])
                             : "memory");
            fence_proxy_async_smem();
            mbar_arrive(smem_u32(&bars->p_full[slot]));
            float2 ls[4];
#pragma unroll
            for (int q = 0; q < 32; ++q) {
                const float2 p = ElemTraits<T>::to_f2(*reinterpret_cast<const typename ElemTraits<T>::T2*>(&pp[q]));
                ls[q & 3] = q < 4 ? p : add2(ls[q & 3], p);
            }
            ls[0] = add2(add2(ls[0], ls[1]), add2(ls[2], ls[3]));
            if (it.seg_tile() < kSets) l_self = 0.f;
            else if (m != m_l) l_self *= ex2(m_l - m);
            m_l = m;
            l_self += ls[0].x + ls[0].y;
            if (it.t + kSets >= it.seg_end()) {
                volatile float2* lp = l_pub + (j % kSums) * 128 + t;
                lp->x = l_self;
                lp->y = m;
            }
            mbar_arrive(smem_u32(&bars->lpub[j % kSums]));

            if (it.seg_last()) {
                // ---- the segment's partial record: this thread's row of the CTA's 256 columns
                float l_tot = 0.f;
                got = true;
#pragma unroll
                for (int i = 0; i < kSets; ++i)
                    if (it.seg_tile() >= i) {
                        // the set of tile j - i: its sums over the segment end there
                        const int js = j - i;
                        got = got && mbar_wait(smem_u32(&bars->lpub[js % kSums]), (js / kSums) & 1, err, code(kWaitRef));
                        const volatile float2* lp = l_pub + (js % kSums) * 128 + t;
                        l_tot += lp->x * ex2(lp->y - m);
                    }
                got = got && mbar_wait(smem_u32(&bars->pv_done[slot]), phase, err, code(kWaitPV));
                if (!warp_ok(got)) break;
                tc_fence_after();
                const long long at = static_cast<long long>(it.g + w) * 128 + t;
                const bool row_ok = t < it.d.rows;
                float* ml = wk.rec_ml + at * kMl;
                if (row_ok && rank == 0) *reinterpret_cast<float2*>(ml) = make_float2(m, l_tot);
                float f[4];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    f[c] = write_cols(trow + kColO + 64 * c, wk.rec_o + at * 512 + 256 * rank + 64 * c, row_ok);
                if (row_ok) *reinterpret_cast<float4*>(ml + 4 + 4 * rank) = make_float4(f[0], f[1], f[2], f[3]);
                tc_fence_before();
                mbar_arrive(smem_u32(&bars->o_free));
            }
        }
    }

    // ---------------------------------------------------------------- teardown
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(&wk.done[w], 1);   // this CTA's records are written (or, after a failure, the status is)
        // the pair finishes together: no CTA leaves while the other may still address it
        mbar_arrive_remote(mapa(smem_u32(&bars->done), peer));
        mbar_wait_cluster_full(smem_u32(&bars->done), 0, err, code(kWaitTeardown));
        if (*err != 0) {
            // after a failure the peer's partial scores may still be in flight
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 20000ull) {
            }
        }
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tbase, kTmemCols);
}

// ------------------------------------------------------------------------------------- merge

constexpr int kMergeWarps = 8;

constexpr uint64_t kPollNs = 1000000;   // 1 ms

__device__ __forceinline__ int load_done(const int* p) {
    int n;
    asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(n) : "l"(p) : "memory");
    return n;
}

// The plan, which a CTA of any worker has seen, is seen by this warp too. (Both have begun when this kernel
// runs, so this does not wait; the end of their kernel would say the same.)
__device__ __forceinline__ void await_plan(const int* done) {
    if (load_done(done) == 0) pdl_wait();
}

// Waits until the workers w0 .. w1 have written their records (warp-wide). They all run when this kernel does,
// but how long they take goes by the lengths: after kPollNs it is the end of their kernel that is awaited.
__device__ __forceinline__ void await_workers(const int* done, int w0, int w1, int lane) {
    const uint64_t t0 = globaltimer_ns();
    for (int w = w0 + lane; __any_sync(0xffffffffu, w <= w1); w += 32) {
        for (;;) {
            const int n = w <= w1 ? load_done(done + w) : 4;
            if (__all_sync(0xffffffffu, n >= 4)) break;
            if (__any_sync(0xffffffffu, globaltimer_ns() - t0 > kPollNs)) {
                pdl_wait();
                return;
            }
            __nanosleep(64);
        }
    }
    __syncwarp();
}

// One output row per `kWarps` warps: each takes every kWarps-th record of the row's groups, keeping
// the running maximum, sum and weighted latent in fp32; the warps meet in shared memory. A row starts
// as soon as the workers of its own records are done, beside those that still work.
template <typename T, int kWarps>
__global__ void __launch_bounds__(32 * kMergeWarps) prefix_merge_kernel(const __grid_constant__ PrefixArgs A, const Work wk) {
    constexpr int kRows = kMergeWarps / kWarps;   // rows per block
    __shared__ float sh_o[kWarps > 1 ? kMergeWarps : 1][512];
    __shared__ float2 sh_ml[kMergeWarps];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int sub = warp % kWarps;
    const int f = blockIdx.x * kRows + warp / kWarps;
    const bool live = f < A.B * A.H;
    float m = -INFINITY, l = 0.f;
    float o[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = 0.f;
    await_plan(wk.done + blockIdx.x % wk.W);
    bool bad = __ldcg(wk.unsorted) != 0;
    if (live && !bad) {
        const int b = f / A.H, h = f % A.H;
        // the row's groups: its request's, and unless that holds the prefix too, its prefix group's
        const int2 rq = wk.fold ? make_int2(-1, 0) : wk.request[b];
        Pieces piece[2];
        piece[0] = wk.pieces[b * ceil_div(A.H, 128) + h / 128];
        piece[1].g = -1;
        if (rq.x >= 0) piece[1] = wk.pieces[rq.x + (f - rq.y) / 128];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (piece[k].g < 0) continue;
            const int g = piece[k].g, w1 = piece[k].w1, r = k == 0 ? h % 128 : (f - rq.y) % 128;
            await_workers(wk.done, piece[k].w0, w1, lane);
            bad = bad || *static_cast<volatile int*>(wk.status) != 0 || __ldcg(wk.bad + g) != 0;
            constexpr int kAhead = 4;
            for (int w = piece[k].w0 + sub; w <= w1; w += kWarps * kAhead) {
                uint4 v[kAhead][2];
                float2 ml[kAhead], fs[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i)
                    if (w + i * kWarps <= w1) {
                        const long long at = static_cast<long long>(g + w + i * kWarps) * 128 + r;
                        ml[i] = __ldcg(reinterpret_cast<const float2*>(wk.rec_ml + at * kMl));
                        fs[i] = make_float2(__ldcg(wk.rec_ml + at * kMl + 4 + lane / 8), __ldcg(wk.rec_ml + at * kMl + 8 + lane / 8));
                        const uint4* src = reinterpret_cast<const uint4*>(wk.rec_o + at * 512);
                        v[i][0] = __ldcg(src + lane);
                        v[i][1] = __ldcg(src + 32 + lane);
                    }
#pragma unroll
                for (int i = 0; i < kAhead; ++i)
                    if (w + i * kWarps <= w1) {
                        const float top = fmaxf(m, ml[i].x);
                        const float a = ex2(m - top), e0 = ex2(ml[i].x - top);
                        const float c2[2] = {e0 * fs[i].x, e0 * fs[i].y};
                        m = top;
                        l = l * a + e0 * ml[i].y;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const uint32_t x[4] = {v[i][q].x, v[i][q].y, v[i][q].z, v[i][q].w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 y = floats_of(x[e]);
                                o[8 * q + 2 * e] = o[8 * q + 2 * e] * a + c2[q] * y.x;
                                o[8 * q + 2 * e + 1] = o[8 * q + 2 * e + 1] * a + c2[q] * y.y;
                            }
                        }
                    }
            }
        }
    }
    if constexpr (kWarps > 1) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) sh_o[warp][256 * q + 8 * lane + e] = o[8 * q + e];
        if (lane == 0) sh_ml[warp] = make_float2(m, l);
        __syncthreads();
        const int first = warp - sub;
        float top = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) top = fmaxf(top, sh_ml[first + i].x);
        float c[kWarps];
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            c[i] = sh_ml[first + i].x == -INFINITY ? 0.f : ex2(sh_ml[first + i].x - top);
            l += c[i] * sh_ml[first + i].y;
        }
        // each warp finishes its share of the columns
        T* out = static_cast<T*>(A.out) + static_cast<long long>(f) * 512;
        if (live)
            for (int x = sub * 32 + lane; x < 512; x += 32 * kWarps) {
                float y = 0.f;
#pragma unroll
                for (int i = 0; i < kWarps; ++i) y += c[i] * sh_o[first + i][x];
                out[x] = ElemTraits<T>::from_f(bad ? NAN : (l == 0.f ? 0.f : y / l));
            }
    } else if (live) {
        const float inv = bad ? NAN : (l == 0.f ? 0.f : 1.f / l);
        uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(A.out) + static_cast<long long>(f) * 512);
#pragma unroll
        for (int q = 0; q < 2; ++q)
            out[32 * q + lane] = make_uint4(pair_of<T>(o[8 * q] * inv, o[8 * q + 1] * inv), pair_of<T>(o[8 * q + 2] * inv, o[8 * q + 3] * inv),
                                            pair_of<T>(o[8 * q + 4] * inv, o[8 * q + 5] * inv), pair_of<T>(o[8 * q + 6] * inv, o[8 * q + 7] * inv));
    }
    pdl_wait();   // this kernel ends after the one before it
}

// ------------------------------------------------------------------------------------- host

struct Layout {
    long long groups;     // most groups
    size_t off_group, off_start, off_pieces, off_request, off_base, off_bad, off_done, off_sum, off_ml, off_o, total;
    int W, own, fold;
};

Layout layout(const PrefixArgs& A, int sms) {
    Layout L = {};
    L.fold = A.H % 128 == 0;
    L.own = A.B * ceil_div(A.H, 128);
    // rows of a prefix group end inside a tile at most once a group
    L.groups = L.own + (L.fold ? 0 : static_cast<long long>(A.B) * A.H / 128 + (A.P < A.B ? A.P : A.B));
    L.W = sms / 2 > 0 ? sms / 2 : 1;
    if (L.W > kMaxWorkers) L.W = kMaxWorkers;
    const size_t groups = static_cast<size_t>(L.groups), recs = groups + L.W;
    size_t off = 256;     // status, unsorted
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off = (off + bytes + 255) / 256 * 256;
        return at;
    };
    L.off_group = take(sizeof(Group) * groups);
    L.off_start = take(sizeof(Start) * L.W);
    L.off_pieces = take(sizeof(Pieces) * groups);
    L.off_request = take(sizeof(int2) * A.B);
    L.off_base = take(sizeof(int) * A.P);
    L.off_bad = take(sizeof(int) * groups);
    L.off_done = take(sizeof(int) * L.W);
    L.off_sum = take(sizeof(float2) * 2 * L.W * kSums * 128);
    L.off_ml = take(recs * 128 * kMl * sizeof(float));
    L.off_o = take(recs * 128 * 512 * 2);
    L.total = off;
    return L;
}

template <typename T>
cudaError_t launch(const PrefixArgs& A, unsigned char* ws, int sms, cudaStream_t s) {
    const Layout L = layout(A, sms);
    Work wk;
    wk.status = reinterpret_cast<int*>(ws);
    wk.unsorted = wk.status + 1;
    wk.group = reinterpret_cast<Group*>(ws + L.off_group);
    wk.start = reinterpret_cast<Start*>(ws + L.off_start);
    wk.pieces = reinterpret_cast<Pieces*>(ws + L.off_pieces);
    wk.request = reinterpret_cast<int2*>(ws + L.off_request);
    wk.gbase = reinterpret_cast<int*>(ws + L.off_base);
    wk.bad = reinterpret_cast<int*>(ws + L.off_bad);
    wk.done = reinterpret_cast<int*>(ws + L.off_done);
    wk.rec_ml = reinterpret_cast<float*>(ws + L.off_ml);
    wk.rec_o = reinterpret_cast<uint16_t*>(ws + L.off_o);
    wk.rowsum = reinterpret_cast<float2*>(ws + L.off_sum);
    wk.W = L.W;
    wk.own = L.own;
    wk.fold = L.fold;
    // the latent as 8 blocks of 64 columns and the rope key as 8 of 8: one load brings a CTA's four
    CUtensorMap lat, rope;
    const uint64_t rows = static_cast<uint64_t>(A.kv_rows), pitch = static_cast<uint64_t>(A.stride) * 2;
    const uint64_t ld[3] = {64, rows, 8}, ls[2] = {pitch, 128}, rd[3] = {8, rows, 8}, rs[2] = {pitch, 16};
    const uint32_t lb[3] = {64, kTile, 4}, rb[3] = {8, kTile, 4};
    if (!encode_tmap_16b(&lat, A.kv, 3, ld, ls, lb, CU_TENSOR_MAP_SWIZZLE_128B) ||
        !encode_tmap_16b(&rope, static_cast<const unsigned char*>(A.kv) + 1024, 3, rd, rs, rb, CU_TENSOR_MAP_SWIZZLE_NONE))
        return cudaErrorInvalidValue;
    cudaError_t e = ensure_dynamic_smem(reinterpret_cast<const void*>(prefix_attend_kernel<T>), static_cast<int>(kSmemBytes));
    if (e != cudaSuccess) return e;
    prefix_plan_kernel<<<1, L.groups <= 256 ? 256 : kPlanThreads, 0, s>>>(A, wk);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * L.W);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if ((e = cudaLaunchKernelEx(&cfg, prefix_attend_kernel<T>, lat, rope, A, wk)) != cudaSuccess) return e;
    cfg.dynamicSmemBytes = 0;
    cfg.blockDim = dim3(32 * kMergeWarps);
    const int out_rows = A.B * A.H;
    // few rows have many records each (a row's group spans up to W workers): 8 warps a row
    if (out_rows <= 4 * sms) {
        cfg.gridDim = dim3(out_rows);
        e = cudaLaunchKernelEx(&cfg, prefix_merge_kernel<T, kMergeWarps>, A, wk);
    } else {
        cfg.gridDim = dim3(ceil_div(out_rows, kMergeWarps));
        e = cudaLaunchKernelEx(&cfg, prefix_merge_kernel<T, 1>, A, wk);
    }
    count_launches(3);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

// The most tiles and fixed costs of groups that the plan may count for these bounds of the lengths.
static long long most_tiles(const PrefixArgs& A) {
    const long long ptiles = (static_cast<long long>(A.max_plen) + kTile - 1) / kTile,
                    otiles = (static_cast<long long>(A.max_len) + kTile - 1) / kTile;
    const long long own = static_cast<long long>(A.B) * ceil_div(A.H, 128),
                    shared = A.H % 128 == 0 ? own : static_cast<long long>(A.B) * A.H / 128 + (A.P < A.B ? A.P : A.B);
    return own * (otiles + kGroupCost) + shared * (ptiles + kGroupCost);
}

bool prefix_sm100_supported(const PrefixArgs& A) {
    auto is16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    return A.dc == 512 && A.dR == 64 && A.stride % 8 == 0 && A.stride <= (1 << 30) && is16(A.kv) && is16(A.qa) &&
           is16(A.qr) && is16(A.out) && A.kv_rows < (1ll << 31) - 4 * kTile &&
           most_tiles(A) < 0x7ff00000ll;   // counted in 32 bits, with the groups' fixed costs
}

size_t prefix_sm100_workspace(const PrefixArgs& A, int sms) { return layout(A, sms).total; }

cudaError_t launch_prefix_sm100(const PrefixArgs& A, bool bf16, void* workspace, int sms, cudaStream_t s) {
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    return bf16 ? launch<__nv_bfloat16>(A, ws, sms, s) : launch<__half>(A, ws, sms, s);
}

}  // namespace mla
