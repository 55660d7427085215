// Arguments and launchers of the serving operators around the decode (append with rotation,
// shared-prefix decode, projection with adapters), shared by their kernels and the C entry points
// in ops_api.cu.
#pragma once
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

#include "latent_attn_b200/mla.h"

namespace mla {

// append_rope.cu. Strides are in elements.
struct AppendRope {
    int B, tokens, H, dc, dR;
    void* kv;
    long long stride, kv_rows;
    const void* c;            // (tokens, dc)
    const void* k;            // (tokens, dR)
    long long c_stride, k_stride;
    const void* w;            // (dc,) norm weight, or null: no norm
    float eps;
    const int* cu;            // (B + 1,) first token of each sequence
    const int* lens;          // (B,) rows already in the cache
    int max_len;
    const int64_t* offs;      // (B,) first cache row, or null: b * max_len
    const int* pages;         // (B, max_pages), or null
    int page_rows, max_pages;
    const float* cos;         // (>= max_len, dR / 2) tables, or null: computed from freq
    const float* sin;
    float freq[64];           // theta^(-2i/dR), rounded to fp32 (dR <= 128)
    const void* q;            // (tokens, H, dR) or null
    void* qo;
    long long q_ts, q_hs, qo_ts, qo_hs;   // token and head strides
    int* new_lens;            // (B,) or null
    int* status;              // bit 0: a token without a place; bit 1: a row outside the cache
};
cudaError_t launch_append_rope(const AppendRope& A, bool bf16, cudaStream_t s);

// prefix_decode.cu / prefix_sm100.cu: decode attention over [the group's prefix | the request's rows].
struct PrefixArgs {
    int B, H, P, dc, dR;
    const void* kv;           // cache rows [latent | rotated rope key]
    long long stride, kv_rows;
    const void* qa;           // (B, H, dc)
    const void* qr;           // (B, H, dR), rotated
    const int* starts;        // (P + 1,) first request of each group
    const int* plens;         // (P,)
    int max_plen;
    const int64_t* poffs;     // (P,) first cache row, or null with ptable
    const int* ptable;        // (P, max_ppages)
    int max_ppages;
    const int* lens;          // (B,)
    int max_len;
    const int64_t* offs;      // (B,) or null with table
    const int* table;         // (B, max_pages)
    int max_pages;
    int page_rows;            // 0: contiguous (poffs, offs)
    float scale;
    void* out;                // (B, H, dc)
};
// CUDA cores, any dimensions: no workspace
cudaError_t launch_prefix_simt(const PrefixArgs& A, bool bf16, cudaStream_t s);
// tensor cores (sm_100): dc 512, dR 64, 16-byte rows and pointers
bool prefix_sm100_supported(const PrefixArgs& A);
size_t prefix_sm100_workspace(const PrefixArgs& A, int sms);
cudaError_t launch_prefix_sm100(const PrefixArgs& A, bool bf16, void* workspace, int sms, cudaStream_t s);

// lora.cu: Y = X W^T + scale_a (X A_a^T) B_a^T, a the token's adapter
struct LoraArgs {
    int M, N, K;
    const void* x;            // (M, K)
    long long x_stride;
    const void* w;            // (N, K)
    int adapters, rank;
    const void* a;            // (adapters, rank, K)
    const void* b;            // (adapters, N, rank)
    const int* ids;           // (M,) adapter of each token; outside [0, adapters): none
    const float* scales;      // (adapters,) or null: 1
    void* y;                  // (M, N)
};
size_t lora_workspace(int M, int N, int K, int adapters, int rank, int sms);
cudaError_t launch_lora(const LoraArgs& A, bool bf16, void* workspace, int sms, cudaStream_t s);

// ---- shared with mla_api.cu: the thread's error message and the device's properties
mla_status_t api_fail(mla_status_t s, const char* fmt, ...);
mla_status_t api_cuda_fail(cudaError_t e, const char* what);   // NO_DEVICE_CODE or CUDA
mla_status_t api_check_config(const mla_config_t* cfg);
bool api_device(int* sms, int* major);

}  // namespace mla
