// paged.h -- parameter blocks, launchers and device helpers of the paged K/V
// cache (layout: include/mugen_attn_paged.h).
#pragma once
#include "common.h"
#include "kernels.h"
#include "mugen_attn_paged.h"

namespace mugen_attn {

struct PagedStore {
    uint8_t* k;  // 16-bit rows or E4M3 codes
    uint8_t* v;
    uint8_t* k_exp;
    uint8_t* v_exp;
    uint16_t* tail_k;
    uint16_t* tail_v;
    uint16_t* k_range;
    const int32_t* table;
    int64_t table_stride;
    int64_t tail_stride;
    int n_pages;
    int p_shift;  // log2(page_tokens)
    int ring;
    int Hk;
    int max_T;
};

// turns per position of each rotated pair: frequency / (2 pi), in 64 bits (passed
// by value: head_dim / 2 of them)
template <int N>
struct RopeTurns {
    double f[N];
};

struct PagedAppendParams {
    PagedStore st;
    const uint16_t* k_new;
    const uint16_t* v_new;
    const uint16_t* q;
    uint16_t* q_out;
    const int32_t* seq_lens;
    const int32_t* new_lens;
    int32_t* seq_lens_out;
    int64_t k_stride, v_stride, q_stride;
    int n_seq;
    int n_new;
    int H;         // query heads rotated (0: none)
    int rope_dim;
    int heads_per_thread;
    int row_blocks;   // workgroups of row work, ahead of the page jobs
    int pages;        // page jobs per (sequence, kv head, tensor): the pages n_new tokens can touch
};

struct PagedDecodeParams {
    PagedStore st;
    const uint16_t* q;
    void* out;
    const int32_t* seq_lens;  // null: every sequence holds fixed_T tokens
    const int32_t* q_lens;
    const int32_t* sel;       // page lists (LIST kernels)
    int n_sel;
    int fixed_T;
    int B;       // sequences (LIST: queries, sequence = item / q_len)
    int q_len;
    int H;
    int G;
    int nrb;     // row blocks per (sequence, kv head)
    int out_dt;
    int chunk;   // tokens per split (0: planned from the device lengths for at most `budget` items)
    int num_splits;
    int budget;
    float scale_log2;
    float r_mult, r_nrb, r_G, r_q_len;  // 1 / (Hk * nrb), 1 / nrb, ... for div_f
    float* ws_o;   // [B][q_len][H][num_splits][D] unnormalised partial outputs
    float* ws_ml;  // [..][2] (max in log2 units, sum)
    int* plan;
};

// most splits of a range
constexpr int kPagedMaxSplits = 128;
// waves that the registers of a SIMD hold: operands of a tile and of the next one
// (8-bit: half the bytes), O and q
__host__ __device__ constexpr int paged_waves_per_simd(int D, bool bits8) {
    return D == 256 ? 1 : D == 128 ? (bits8 ? 3 : 2) : (bits8 ? 4 : 3);
}
// A workgroup: WR waves take a tile's 16-row blocks side by side, paged_tiles tiles
// are under way.  4 waves in all, one to a SIMD, or 12 (three row blocks), which
// fill a CU that holds 3 to a SIMD (two workgroups of 6 do not fit beside each other:
// 2, 2, 1, 1 waves each; 5 drafted tokens of 28 / 4 heads over 4 x 31k 46.7 -> 37.7 us)
__host__ __device__ constexpr int paged_tiles(int D, bool bits8, int WR) {
    return WR == 1 ? 4 : WR == 2 ? 2 : WR == 4 ? 1 : paged_waves_per_simd(D, bits8) >= 3 ? 4 : 2;
}
__host__ __device__ constexpr int paged_groups_per_cu(int D, bool bits8, int WR) {
    const int waves = WR * paged_tiles(D, bits8, WR), most = 4 * paged_waves_per_simd(D, bits8);
    return waves > 4 ? 1 : most / 4;
}

struct PageSelectParams {
    PagedStore st;
    const uint16_t* q;
    int32_t* pages;
    const int32_t* seq_lens;
    const int32_t* q_lens;
    int B, q_len, H, G;
    int n_select, n_first, n_last;
    int max_pages;   // row stride of the scores
    uint64_t* keys;  // [B][q_len][Hk][max_pages]: the scores as integers of the same order
};

struct PagedGatherParams {
    PagedStore st;
    uint16_t* k_out;  // [T][Hk * D]
    uint16_t* v_out;
    int seq;
    int T;
    int v16;  // V in fp16 whatever the store's type
};

hipError_t launch_paged_append(PagedAppendParams p, const RopeTurns<128>& turns, int D, int dt, bool bits8, hipStream_t st, KernelTimer* t);
hipError_t launch_paged_gather(const PagedGatherParams& p, int D, int dt, bool bits8, hipStream_t st, KernelTimer* t);
// wr: 16-row blocks of one workgroup (1 .. 4; 1, 2 or 4 at head_dim 256)
hipError_t launch_paged_decode16(const PagedDecodeParams& p, int nwg, int D, int dt, int wr, hipStream_t st,
                                 KernelTimer* t);
hipError_t launch_paged_decode8(const PagedDecodeParams& p, int nwg, int D, int dt, int wr, hipStream_t st,
                                KernelTimer* t);
hipError_t launch_paged_combine(const PagedDecodeParams& p, int D, hipStream_t st, KernelTimer* t);
hipError_t launch_page_score(const PageSelectParams& p, int D, int dt, hipStream_t st, KernelTimer* t);
hipError_t launch_page_select(const PageSelectParams& p, hipStream_t st, KernelTimer* t);

// n / d for 0 <= n < 2^23, rd = 1.0f / d to one ulp (a few instructions instead of
// the 35 of an integer division)
__device__ __forceinline__ int div_f(int n, int d, float rd) {
    const int q = (int)((float)n * rd), r = n - q * d;
    return r < 0 ? q - 1 : r >= d ? q + 1 : q;
}

// the physical page of a table entry, or -1
__device__ __forceinline__ int checked_page(int id, int n_pages) { return (uint32_t)id < (uint32_t)n_pages ? id : -1; }

// E8M0 byte -> 2^(byte - 127) (byte >= 1)
__device__ __forceinline__ float exp_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// two E4M3 codes (the low or the high half of w) times a power of two, in DT
template <int DT, bool HI>
__device__ __forceinline__ uint32_t cvt2_fp8(uint32_t w, float scale) {
    if constexpr (DT == DT_BF16)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
}
// eight codes -> eight 16-bit values
template <int DT>
__device__ __forceinline__ u32x4_t cvt8_fp8(uint32_t lo, uint32_t hi, float scale) {
    return u32x4_t{cvt2_fp8<DT, false>(lo, scale), cvt2_fp8<DT, true>(lo, scale), cvt2_fp8<DT, false>(hi, scale),
                   cvt2_fp8<DT, true>(hi, scale)};
}

}  // namespace mugen_attn
