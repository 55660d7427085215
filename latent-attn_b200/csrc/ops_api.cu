// C entry points of the serving operators: argument checks and launches. As everywhere in the
// library they return status codes, allocate nothing and never synchronise.
#include <cmath>
#include <cstring>

#include "mla_internal.cuh"
#include "ops.cuh"

using mla::api_cuda_fail;
using mla::api_fail;

namespace {

mla_status_t check_dtype(mla_dtype_t d) {
    if (d != MLA_DTYPE_F16 && d != MLA_DTYPE_BF16)
        return api_fail(MLA_ERR_UNSUPPORTED, "dtype must be F16 or BF16 (got %d)", static_cast<int>(d));
    return MLA_OK;
}

// A launch may throw on the host (no memory, a lock): nothing of that crosses a C entry.
template <typename F>
cudaError_t launch(F f) {
    try {
        return f();
    } catch (...) {
        return cudaErrorMemoryAllocation;
    }
}

}  // namespace

extern "C" {

mla_status_t mla_cache_append_rope(const mla_config_t* cfg, const mla_append_rope_args_t* a, mla_stream_t stream) {
    mla_status_t st = mla::api_check_config(cfg);
    if (st != MLA_OK) return st;
    if (!a) return api_fail(MLA_ERR_INVALID_ARGUMENT, "args is null");
    st = check_dtype(a->dtype);
    if (st != MLA_OK) return st;
    const int dc = cfg->kv_lora_rank, dR = cfg->qk_rope_head_dim, H = cfg->num_heads;
    if (dR % 2 != 0 || dR > 256)
        return api_fail(MLA_ERR_UNSUPPORTED, "qk_rope_head_dim must be even and <= 256 (got %d)", dR);
    if (a->batch <= 0) return api_fail(MLA_ERR_INVALID_ARGUMENT, "batch must be positive, got %d", a->batch);
    if (a->tokens < 0) return api_fail(MLA_ERR_INVALID_ARGUMENT, "tokens must be >= 0, got %d", a->tokens);
    if (a->max_seq_len <= 0)
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "max_seq_len must be positive, got %d", a->max_seq_len);
    if (!a->kv_cache || !a->cu_tokens || !a->seq_lens || (a->tokens > 0 && (!a->c || !a->k_rope)))
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "null pointer");
    if (a->kv_total_rows <= 0) return api_fail(MLA_ERR_INVALID_ARGUMENT, "kv_total_rows must be positive");
    if ((a->rope_cos == nullptr) != (a->rope_sin == nullptr))
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "give both rope_cos and rope_sin, or neither (computed angles)");
    if (!a->rope_cos && dR > 2 * mla::kMaxRopeHalf)
        return api_fail(MLA_ERR_UNSUPPORTED, "computed angles need qk_rope_head_dim <= %d (got %d)", 2 * mla::kMaxRopeHalf, dR);
    if (!(a->rope_theta >= 0.f)) return api_fail(MLA_ERR_INVALID_ARGUMENT, "rope_theta must be >= 0");
    if (a->norm_weight && !(a->norm_eps >= 0.f)) return api_fail(MLA_ERR_INVALID_ARGUMENT, "norm_eps must be >= 0");
    if (a->page_table) {
        if (a->kv_offsets) return api_fail(MLA_ERR_INVALID_ARGUMENT, "page_table excludes kv_offsets");
        if (a->page_rows <= 0) return api_fail(MLA_ERR_INVALID_ARGUMENT, "page_rows must be positive, got %d", a->page_rows);
        if (static_cast<long long>(a->max_pages) * a->page_rows < a->max_seq_len)
            return api_fail(MLA_ERR_INVALID_ARGUMENT, "max_pages %d x page_rows %d < max_seq_len %d", a->max_pages,
                            a->page_rows, a->max_seq_len);
    }
    if ((a->q_rope == nullptr) != (a->q_out == nullptr))
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "give q_rope together with q_out");
    if (a->new_lens && a->new_lens == a->seq_lens)
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "new_lens must not be seq_lens (every token reads its sequence's length)");
    mla::AppendRope A;
    std::memset(&A, 0, sizeof(A));
    A.B = a->batch; A.tokens = a->tokens; A.H = H; A.dc = dc; A.dR = dR;
    A.kv = a->kv_cache;
    A.stride = a->kv_row_stride ? a->kv_row_stride : dc + dR;
    A.kv_rows = a->kv_total_rows;
    A.c = a->c; A.k = a->k_rope;
    A.c_stride = a->c_stride ? a->c_stride : dc;
    A.k_stride = a->k_stride ? a->k_stride : dR;
    A.w = a->norm_weight; A.eps = a->norm_eps;
    A.cu = a->cu_tokens; A.lens = a->seq_lens; A.max_len = a->max_seq_len;
    A.offs = a->kv_offsets; A.pages = a->page_table; A.page_rows = a->page_rows; A.max_pages = a->max_pages;
    A.cos = a->rope_cos; A.sin = a->rope_sin;
    A.q = a->q_rope; A.qo = a->q_out;
    A.q_hs = a->q_head_stride ? a->q_head_stride : dR;
    A.q_ts = a->q_token_stride ? a->q_token_stride : static_cast<long long>(H) * dR;
    A.qo_hs = a->q_out_head_stride ? a->q_out_head_stride : dR;
    A.qo_ts = a->q_out_token_stride ? a->q_out_token_stride : static_cast<long long>(H) * dR;
    A.new_lens = a->new_lens; A.status = a->status;
    if (A.stride < dc + dR) return api_fail(MLA_ERR_INVALID_ARGUMENT, "kv_row_stride %lld < d_c + d_R", A.stride);
    if (A.c_stride < 0 || A.k_stride < 0 || A.q_ts < 0 || A.q_hs < 0)
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "strides must be >= 0");
    // output rows must not overlap, whichever of tokens and heads is the outer dimension
    auto apart = [dR](int64_t outer, int64_t inner, int n_inner) {
        return (n_inner == 1 || inner >= dR) && outer >= (n_inner - 1) * (n_inner > 1 ? inner : 0) + dR;
    };
    const bool one_token = a->tokens <= 1;
    if (A.q && !(one_token ? H == 1 || A.qo_hs >= dR
                           : apart(A.qo_ts, A.qo_hs, H) || (H > 1 && apart(A.qo_hs, A.qo_ts, a->tokens))))
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "q_out's rows overlap");
    if (!A.cos) {
        // as mla_decode: the double-precision power rounded once to fp32
        const double theta = a->rope_theta > 0.f ? static_cast<double>(a->rope_theta) : 10000.0;
        for (int i = 0; i < dR / 2; ++i) A.freq[i] = static_cast<float>(std::pow(theta, -2.0 * i / static_cast<double>(dR)));
    }
    const cudaError_t e = launch([&] { return mla::launch_append_rope(A, a->dtype == MLA_DTYPE_BF16, reinterpret_cast<cudaStream_t>(stream)); });
    return e == cudaSuccess ? MLA_OK : api_cuda_fail(e, "append kernel launch");
}

static mla_status_t make_prefix(const mla_config_t* cfg, const mla_prefix_args_t* a, mla::PrefixArgs* A) {
    mla_status_t st = mla::api_check_config(cfg);
    if (st != MLA_OK) return st;
    if (!a) return api_fail(MLA_ERR_INVALID_ARGUMENT, "args is null");
    st = check_dtype(a->dtype);
    if (st != MLA_OK) return st;
    const int dc = cfg->kv_lora_rank, dR = cfg->qk_rope_head_dim, H = cfg->num_heads;
    if (dc % 32 != 0 || dc > 1024)
        return api_fail(MLA_ERR_UNSUPPORTED, "kv_lora_rank must be a multiple of 32 and <= 1024 (got %d)", dc);
    if (dR % 2 != 0 || dR > 256)
        return api_fail(MLA_ERR_UNSUPPORTED, "qk_rope_head_dim must be even and <= 256 (got %d)", dR);
    if (a->batch <= 0) return api_fail(MLA_ERR_INVALID_ARGUMENT, "batch must be positive, got %d", a->batch);
    if (a->num_groups <= 0) return api_fail(MLA_ERR_INVALID_ARGUMENT, "num_groups must be positive, got %d", a->num_groups);
    if (static_cast<long long>(a->batch) * H > (1 << 24))
        return api_fail(MLA_ERR_UNSUPPORTED, "batch x num_heads must be <= 2^24");
    if (a->max_prefix_len < 0 || a->max_seq_len < 0 || a->max_prefix_len > (1 << 29) || a->max_seq_len > (1 << 29))
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "max_prefix_len and max_seq_len must be in [0, 2^29]");
    if (!a->kv_cache || !a->q_absorbed || !a->q_rope || !a->group_starts || !a->prefix_lens || !a->seq_lens || !a->output)
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "null pointer");
    if (a->kv_total_rows <= 0) return api_fail(MLA_ERR_INVALID_ARGUMENT, "kv_total_rows must be positive");
    const int64_t stride = a->kv_row_stride ? a->kv_row_stride : dc + dR;
    if (stride < dc + dR) return api_fail(MLA_ERR_INVALID_ARGUMENT, "kv_row_stride %lld < d_c + d_R", (long long)stride);
    if (!(a->softmax_scale >= 0.f) || std::isinf(a->softmax_scale))
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "softmax_scale must be finite and >= 0");
    if (a->page_rows < 0 || a->page_rows % 64 != 0)
        return api_fail(MLA_ERR_UNSUPPORTED, "page_rows must be a multiple of 64, got %d", a->page_rows);
    if (a->page_rows > 0) {
        if (a->kv_offsets || a->prefix_offsets)
            return api_fail(MLA_ERR_INVALID_ARGUMENT, "page_rows excludes kv_offsets and prefix_offsets");
        if ((a->max_prefix_len > 0 && !a->prefix_table) || (a->max_seq_len > 0 && !a->page_table))
            return api_fail(MLA_ERR_INVALID_ARGUMENT, "page_rows needs prefix_table and page_table");
        if (static_cast<long long>(a->max_prefix_pages) * a->page_rows < a->max_prefix_len ||
            static_cast<long long>(a->max_pages) * a->page_rows < a->max_seq_len)
            return api_fail(MLA_ERR_INVALID_ARGUMENT, "a page table has fewer pages than its max length needs");
    } else if (a->page_table || a->prefix_table) {
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "page tables need page_rows");
    } else if ((a->max_prefix_len > 0 && !a->prefix_offsets) || (a->max_seq_len > 0 && !a->kv_offsets)) {
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "give prefix_offsets and kv_offsets, or page tables with page_rows");
    }
    if (a->kernel < MLA_KERNEL_AUTO || a->kernel > MLA_KERNEL_CUDA_CORE)
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "unknown kernel %d", a->kernel);
    std::memset(A, 0, sizeof(*A));
    A->B = a->batch; A->H = H; A->P = a->num_groups; A->dc = dc; A->dR = dR;
    A->kv = a->kv_cache; A->stride = stride; A->kv_rows = a->kv_total_rows;
    A->qa = a->q_absorbed; A->qr = a->q_rope;
    A->starts = a->group_starts;
    A->plens = a->prefix_lens; A->max_plen = a->max_prefix_len; A->poffs = a->prefix_offsets;
    A->ptable = a->prefix_table; A->max_ppages = a->max_prefix_pages;
    A->lens = a->seq_lens; A->max_len = a->max_seq_len; A->offs = a->kv_offsets;
    A->table = a->page_table; A->max_pages = a->max_pages; A->page_rows = a->page_rows;
    A->scale = a->softmax_scale > 0.f ? a->softmax_scale : 1.0f / std::sqrt(static_cast<float>(cfg->qk_nope_head_dim + dR));
    A->out = a->output;
    return MLA_OK;
}

// Which kernel serves the call: the tensor cores' wherever their shape and alignment rules hold.
static mla_status_t choose_prefix(const mla_prefix_args_t* a, const mla::PrefixArgs& A, bool* tc, int* sms) {
    int major = 0;
    if (!mla::api_device(sms, &major)) return api_fail(MLA_ERR_CUDA, "no CUDA device");
    const bool can = major == 10 && mla::prefix_sm100_supported(A);
    if (a->kernel == MLA_KERNEL_TENSOR_CORE && !can)
        return api_fail(MLA_ERR_UNSUPPORTED, "the tensor-core kernel needs sm_100, kv_lora_rank 512, qk_rope_head_dim 64 "
                        "and 16-byte aligned rows");
    *tc = can && a->kernel != MLA_KERNEL_CUDA_CORE;
    return MLA_OK;
}

mla_status_t mla_prefix_decode_workspace_size(const mla_config_t* cfg, const mla_prefix_args_t* a, size_t* bytes) {
    mla::PrefixArgs A;
    bool tc = false;
    int sms = 0;
    mla_status_t st = make_prefix(cfg, a, &A);
    if (st == MLA_OK) st = choose_prefix(a, A, &tc, &sms);
    if (st != MLA_OK) return st;
    if (!bytes) return api_fail(MLA_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = tc ? mla::prefix_sm100_workspace(A, sms) : 0;
    return MLA_OK;
}

mla_status_t mla_prefix_decode(const mla_config_t* cfg, const mla_prefix_args_t* a, void* workspace,
                               size_t workspace_bytes, mla_stream_t stream) {
    mla::PrefixArgs A;
    bool tc = false;
    int sms = 0;
    mla_status_t st = make_prefix(cfg, a, &A);
    if (st == MLA_OK) st = choose_prefix(a, A, &tc, &sms);
    if (st != MLA_OK) return st;
    const bool bf16 = a->dtype == MLA_DTYPE_BF16;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (tc) {
        const size_t need = mla::prefix_sm100_workspace(A, sms);
        if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
            return api_fail(MLA_ERR_WORKSPACE, "workspace is null or not 256-byte aligned");
        if (workspace_bytes < need) return api_fail(MLA_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);
        e = launch([&] { return mla::launch_prefix_sm100(A, bf16, workspace, sms, s); });
    } else {
        e = launch([&] { return mla::launch_prefix_simt(A, bf16, s); });
    }
    return e == cudaSuccess ? MLA_OK : api_cuda_fail(e, "prefix decode kernel launch");
}

static mla_status_t make_lora(const mla_lora_args_t* a, mla::LoraArgs* A, int* sms) {
    if (!a) return api_fail(MLA_ERR_INVALID_ARGUMENT, "args is null");
    const mla_status_t st = check_dtype(a->dtype);
    if (st != MLA_OK) return st;
    if (a->M <= 0 || a->N <= 0 || a->K <= 0)
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "M, N and K must be positive (M=%d, N=%d, K=%d)", a->M, a->N, a->K);
    if (a->num_adapters <= 0) return api_fail(MLA_ERR_INVALID_ARGUMENT, "num_adapters must be positive, got %d", a->num_adapters);
    if (a->K % 8 != 0 || a->x_stride % 8 != 0)
        return api_fail(MLA_ERR_UNSUPPORTED, "K and x_stride must be multiples of 8 (K=%d, x_stride=%lld)", a->K, (long long)a->x_stride);
    if (a->rank <= 0 || a->rank % 8 != 0 || a->rank > 256)
        return api_fail(MLA_ERR_UNSUPPORTED, "rank must be a multiple of 8 and <= 256 (got %d)", a->rank);
    if (a->M > (1 << 23) || a->N > (1 << 28)) return api_fail(MLA_ERR_UNSUPPORTED, "M must be <= 2^23 and N <= 2^28");
    // rows of the intermediate A_a X[m] (per 256 tokens, adapter and 64 ranks), counted in 32 bits
    if ((a->M + 255ll) * (a->num_adapters < 256 ? a->num_adapters : 256) * ((a->rank + 63) / 64) > 0x7fffffffll)
        return api_fail(MLA_ERR_UNSUPPORTED, "too many tokens for %d adapters of rank %d (M=%d)", a->num_adapters, a->rank, a->M);
    if (!a->X || !a->W || !a->lora_a || !a->lora_b || !a->adapter_ids || !a->Y)
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "null pointer");
    if (a->x_stride != 0 && a->x_stride < a->K) return api_fail(MLA_ERR_INVALID_ARGUMENT, "x_stride %lld < K", (long long)a->x_stride);
    if ((reinterpret_cast<uintptr_t>(a->X) | reinterpret_cast<uintptr_t>(a->W) | reinterpret_cast<uintptr_t>(a->lora_a) |
         reinterpret_cast<uintptr_t>(a->lora_b)) % 16 != 0)
        return api_fail(MLA_ERR_INVALID_ARGUMENT, "X, W, lora_a and lora_b must be 16-byte aligned");
    int major = 0;
    if (!mla::api_device(sms, &major)) return api_fail(MLA_ERR_CUDA, "no CUDA device");
    if (major != 10) return api_fail(MLA_ERR_NO_DEVICE_CODE, "mla_linear_lora needs an sm_100 GPU");
    *A = {a->M, a->N, a->K, a->X, a->x_stride ? a->x_stride : a->K, a->W, a->num_adapters, a->rank,
          a->lora_a, a->lora_b, a->adapter_ids, a->scales, a->Y};
    return MLA_OK;
}

mla_status_t mla_linear_lora_workspace_size(const mla_lora_args_t* a, size_t* bytes) {
    mla::LoraArgs A;
    int sms = 0;
    const mla_status_t st = make_lora(a, &A, &sms);
    if (st != MLA_OK) return st;
    if (!bytes) return api_fail(MLA_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = mla::lora_workspace(A.M, A.N, A.K, A.adapters, A.rank, sms);
    return MLA_OK;
}

mla_status_t mla_linear_lora(const mla_lora_args_t* a, void* workspace, size_t workspace_bytes, mla_stream_t stream) {
    mla::LoraArgs A;
    int sms = 0;
    const mla_status_t st = make_lora(a, &A, &sms);
    if (st != MLA_OK) return st;
    const size_t need = mla::lora_workspace(A.M, A.N, A.K, A.adapters, A.rank, sms);
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
        return api_fail(MLA_ERR_WORKSPACE, "workspace is null or not 256-byte aligned");
    if (workspace_bytes < need) return api_fail(MLA_ERR_WORKSPACE, "workspace too small: %zu < %zu bytes", workspace_bytes, need);
    const cudaError_t e = launch([&] {
        return mla::launch_lora(A, a->dtype == MLA_DTYPE_BF16, workspace, sms, reinterpret_cast<cudaStream_t>(stream));
    });
    return e == cudaSuccess ? MLA_OK : api_cuda_fail(e, "projection with adapters: kernel launch");
}

}  // extern "C"
