// Host-side launchers of the vlb200 kernels (implemented in vlb_kernels.cu).
#pragma once

#include <cuda_runtime.h>

#include "vlb_internal.cuh"

namespace vlb {

cudaError_t launch_dequant(const DevMat& m, const Grids& g, float* out, cudaStream_t s);
cudaError_t launch_gemv(const DevMat& m, const Grids& g, const float* x, uint32_t ntok,
                        uint32_t xstride, float* y, uint32_t ystride, cudaStream_t s);
// logits[t][e] = f32(sequential f64 sum of xd[t][c] * wd[e][c]), scores = score function of them;
// xd / wd are the f64 widenings of the f32 activations / router weights (H % 2 == 0)
cudaError_t launch_router(const double* xd, const double* wd, uint32_t T, uint32_t H, uint32_t E, int score,
                          float* logits, float* scores, cudaStream_t s);
cudaError_t launch_widen(const float* src, size_t n, double* dst, cudaStream_t s);
// per-token max|x| bits; with xd non-null also the rows widened to f64
cudaError_t launch_prescale(const float* x, uint32_t T, uint32_t H, uint32_t* xmax, double* xd, cudaStream_t s);
cudaError_t launch_scores(const float* logits, size_t n, int score, float* scores,
                          cudaStream_t s);
cudaError_t launch_route(const float* scores, const float* bias, const uint32_t* token_ids,
                         const uint32_t* tid2eid, uint32_t vocab, uint32_t T, uint32_t E,
                         uint32_t k, int score, int hash_routing, float route_scale,
                         uint32_t* idx, float* weights, uint32_t* error_flag, cudaStream_t s);
// The whole layer: routing, dispatch, gate/up + SwiGLU, down, combine (the expert products on the
// decode kernels, or on the prefill kernels when p.prefill is set).
// ev: optional 6 events recorded at the phase boundaries (start, routed, dispatched, gate/up done,
// down done, combined).
constexpr int kMoePhases = 5;
cudaError_t launch_moe(const MoeParams& p, cudaStream_t s, cudaEvent_t* ev = nullptr);
// Prefill path (vlb_prefill.cu): column-tile plan after dispatch, then the tcgen05 grouped GEMMs
// (each preceded by the fp16 conversion of its activations).
uint32_t prefill_max_tiles(uint32_t T, uint32_t k, uint32_t E);
uint32_t prefill_box_rows();  // rows of the B operand's TMA box
cudaError_t launch_prefill_plan(const MoeParams& p, cudaStream_t s);
cudaError_t launch_prefill_gateup(const MoeParams& p, unsigned grid, cudaStream_t s);
cudaError_t launch_prefill_down(const MoeParams& p, unsigned grid, cudaStream_t s);
cudaError_t launch_stable_sort(const MoeParams& p, cudaStream_t s);
// Decode path (vlb_decode.cu): IQ2_XXS / Q8_0 expert products on mma.sync fed by a bulk-copy ring,
// one CTA per SM.
cudaError_t launch_decode_gateup(const MoeParams& p, unsigned n_sms, cudaStream_t s);
// fmt_bit set of the storage types the decode kernel of a phase serves: Q8_0 and the phase's IQ
// type (IQ2_XXS before IQ1_S before IQ3_XXS when several are present) if its stage carve fits
uint32_t decode_ring_types(const MoeParams& p, bool gateup);
cudaError_t launch_decode_down(const MoeParams& p, unsigned n_sms, cudaStream_t s);
// Expert-parallel helpers (vlb_ep.cu)
cudaError_t launch_ep_validate(const uint32_t* idx, size_t n, uint32_t E, uint32_t* flag, cudaStream_t s);
// expert ids -> exchange slots (slot_of null: identity); out-of-range ids flagged and replaced by 0
cudaError_t launch_ep_slots(const uint32_t* idx, size_t n, uint32_t E, const uint32_t* slot_of, uint32_t* out,
                            uint32_t* flag, cudaStream_t s);
// f32 rows -> fp16 rows with a per-row power-of-two scale (scale[r] = the inverse factor)
cudaError_t launch_ep_pack_half(const float* y, uint32_t rows, uint32_t H, __half* out, float* scale, cudaStream_t s);
cudaError_t launch_ep_combine_half(const __half* rows, const float* scale, const uint32_t* elem_row, uint32_t T,
                                   uint32_t k, const float* shared_rows, uint32_t H, float* out, cudaStream_t s);
cudaError_t launch_ep_gather(const uint32_t* pair_token, const uint32_t* pair_slot, const uint32_t* idx,
                             uint32_t n, uint32_t k, uint32_t epr, const float* x, uint32_t H, float* send_x,
                             uint32_t* send_expert, cudaStream_t s);
// Half-row exchange: fp16 send rows + (expert, weight, max|x|) meta, and the own tokens' rows.
cudaError_t launch_ep_gather_half(const uint32_t* pair_token, const uint32_t* pair_slot, const uint32_t* idx,
                                  const float* sorted_w, uint32_t n, uint32_t k, uint32_t epr, const float* x,
                                  const uint32_t* xmax, uint32_t H, __half* rows, uint32_t* meta, cudaStream_t s);
cudaError_t launch_ep_own_rows(const float* x, const uint32_t* xmax, uint32_t T, uint32_t H, uint32_t epr,
                               __half* rows, uint32_t* meta, cudaStream_t s);
cudaError_t launch_ep_combine(const float* y, const uint32_t* elem_row, uint32_t T, uint32_t k,
                              const float* shared_rows, uint32_t H, float* out, cudaStream_t s);
// RMSNorm rows (bit-exact); xmax non-null: also each row's max|out| bits; out_d: the rows as f64.
// width % 4 == 0 and
// width <= kRmsMaxWidth (the row is staged in shared memory).
constexpr uint32_t kRmsMaxWidth = 24576;  // the row staged as f64 in shared memory
// Whether the Hyper-Connection entry kernel's shared-memory plan fits m copies of a hidden row.
bool hc_entry_fits(uint32_t m, uint32_t H);
cudaError_t launch_rms_norm(const float* x, const float* w, uint32_t rows, uint32_t width,
                            float eps, float* out, uint32_t* xmax, double* out_d, cudaStream_t s);

// Launches a kernel that may start before the kernel ahead of it on the stream has ended: its blocks
// come up meanwhile and wait (griddepcontrol.wait) before they touch anything that kernel may write
// or read. Every block waits before it ends, so that a kernel behind waits for all before it.
// cluster: blocks of a cluster, 0 none.
template <typename... P, typename... A>
cudaError_t launch_chained(void (*kernel)(P...), dim3 grid, uint32_t block, size_t smem, uint32_t cluster, cudaStream_t s,
                           const A&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    if (cluster) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// ---- products on 8-bit integers (vlb_int8.cu) ----
struct Int8QuantParams {
    const void* x;             // rows of VLB_DTYPE_F32 / F16 / BF16
    const void* up;            // SwiGLU's second operand (same type and stride), or null
    const uint32_t* row_index; // row r is x's row row_index[r] (none there: zeros), or null
    int8_t* q;
    float* scale;
    size_t x_stride, q_stride; // elements
    uint64_t x_rows;
    uint32_t rows, cols;
    uint32_t fill_cols;        // columns written: cols, then zeros
    float limit;               // SwiGLU clamp, 0: none
};
struct Int8GatherParams {
    const int8_t* x;           // [x_rows] quantized rows of `pitch` bytes (a multiple of 16)
    const float* x_scale;
    const uint32_t* row_index; // an index >= x_rows: a row of zeros, scale 0
    int8_t* q;
    float* scale;
    size_t pitch;
    uint32_t x_rows, rows;
};
struct Int8LinearParams {
    const int8_t* x;           // [rows] of x_stride
    const float* x_scale;
    const float* row_weight;   // or null
    const int8_t* w;           // [groups x out_cols] of w_stride
    const float* w_scale;      // [groups x out_cols]
    const uint32_t* offsets;   // [groups + 1] or null (one group, every row)
    void* y;
    uint32_t* error;           // the handle's word in host memory: 1 once a wait has run out
    size_t x_stride, w_stride, y_stride;
    uint32_t rows, cols, out_cols, groups;
};
constexpr uint32_t kInt8MaxGroups = 1024;
cudaError_t launch_int8_gather(const Int8GatherParams& p, cudaStream_t s);
cudaError_t launch_int8_quantize(const Int8QuantParams& p, int x_type, cudaStream_t s);
// A product of few rows in one launch, its rows quantized on the way (q: their source, x_type I8:
// unused); int8_few: whether it takes the call.
bool int8_few(const Int8LinearParams& l);
cudaError_t launch_int8_few(const Int8LinearParams& l, const Int8QuantParams& q, int x_type, int y_type, cudaStream_t s);
// after_quantize: launch_int8_quantize went before it on the stream (the product may start beside it)
cudaError_t launch_int8_linear(const Int8LinearParams& p, int y_type, bool after_quantize, cudaStream_t s);

// ---- the router's balance loss (vlb_balance.cu) ----
struct BalanceParams {
    const void* logits;
    const uint32_t* idx;         // [T x k]
    const uint8_t* mask;         // [T] or null
    const uint32_t* seq_offsets; // [S + 1] or null (S == 1, every token)
    const float* upstream;       // or null: 1
    float* loss;                 // or null
    uint32_t* counts;            // [S x E]
    void* dlogits;               // or null
    // workspace
    uint32_t* ticket;
    double* partial;             // [kBalanceBlocks] the blocks' losses
    uint32_t* part;              // [S x parts x (E + 1)] counts and live tokens of a sequence's parts
    size_t stride, grad_stride;
    uint32_t T, E, k, S, parts;
    int score, logits_type;
    float coefficient;
};
constexpr uint32_t kBalanceBlocks = 296;  // 2 blocks of 512 threads on each of 148 SMs
constexpr uint32_t kBalOneTokens = 128;   // up to here one block does the whole call
uint32_t balance_parts(uint32_t T, uint32_t S);  // parts of a sequence's counts in the workspace
uint64_t balance_parts_bound(uint32_t T, uint32_t S);  // of all sequences, of the largest call up to T and S
cudaError_t launch_balance(const BalanceParams& p, cudaStream_t s);

}  // namespace vlb
