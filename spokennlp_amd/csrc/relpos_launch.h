// Launch geometry of the relative-position attention kernels (host side).
#pragma once
#include "relpos.h"

int amdseg_relpos_fwd_impl(const RpArgs& a, int dtype, hipStream_t s);
int amdseg_relpos_bwd_impl(const RpArgs& a, int dtype, void* dtable, float* sums, hipStream_t s);

int amdseg_relpos_sums_impl(const float* part, float* sums, int64_t wgs, const int* map, int span, int pad, int buckets, int heads, void* dtable, int bf16,
                            hipStream_t s);
size_t amdseg_relpos_bias_ws_impl(int B, int heads, int Lq, int span);
int amdseg_relpos_bias_fwd_impl(const RpArgs& a, int off, int dtype, hipStream_t s);
int amdseg_relpos_bias_bwd_impl(const void* d, int dtype, const int* map, int span, int buckets, int B, int heads, int Lq, int Lk, int off, float* dtable,
                                float* ws, hipStream_t s);

// dynamic LDS beyond 64 KiB has to be asked for per kernel and device
static inline int rp_allow_lds(const void* kernel, int bytes) {
    if (bytes <= 65536) return 0;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return e == hipSuccess ? 0 : (int)e;
}
// 16-row tiles a wave carries as columns: two (every LDS fragment feeds two products; 32 x 512 forward 54 us against 64, dK / dV 108 against 146) unless one
// gives the CUs a second workgroup that they would not have: grids of up to 256 (2048 rows of 16 heads: dK / dV 73 us against 77), forward and dQ at D <= 64 up
// to 384 (2 x 2048 rows of 12 heads: forward 59 against 66, dQ 64 against 71; dK / dV 122 against 98; at 432 two win: 22 against 22.5, 27 against 31).  fp32: one (registers).
// D > 64 in bf16: two accumulators of 128 columns cost the dK / dV kernel its second wave a SIMD (16 x 512: 113 us against 104 with one tile), and a forward grid of three rounds or more runs better on three waves a SIMD of one tile (4 x 2048:
// 177 against 165).
static inline int rp_qt(int64_t wgs_of_two, int most_of_one, int dtype) { return dtype == 1 ? 1 : wgs_of_two <= most_of_one ? 1 : 2; }
// (packed: a sequence's last block is half full on average)
static inline int64_t rp_blocks_of_two(const RpArgs& a, int L, int T) { return a.cu_q ? (int64_t)(T + 127) / 128 + a.B / 2 : (int64_t)((L + 127) / 128) * a.B; }
static inline int64_t rp_wgs_of_two(const RpArgs& a) { return rp_blocks_of_two(a, a.Lq, a.Tq) * a.heads; }
static inline int rp_dq_qt(const RpArgs& a, int dtype) { return rp_qt(rp_wgs_of_two(a), a.D > 64 ? 256 : 384, dtype); }
static inline int rp_fwd_qt(const RpArgs& a, int dtype) { return a.D > 64 && rp_wgs_of_two(a) >= 768 ? 1 : rp_dq_qt(a, dtype); }
static inline int rp_dkv_qt(const RpArgs& a, int dtype) { return a.D > 64 ? 1 : rp_qt(rp_blocks_of_two(a, a.Lk, a.Tk) * a.kv_heads, 256, dtype); }
// row blocks of a batch (packed: as many as there can be)
static inline int64_t rp_row_blocks(const RpArgs& a, int L, int T, int rows) { return a.cu_q ? (int64_t)T / rows + a.B : (int64_t)((L + rows - 1) / rows) * a.B; }
// how the workgroups of one split are numbered (rp_place, rp_slot): row blocks of `rows` rows, `heads` of them over a.kv_heads.  nmain < 0: too many.  Packed: runs of
// 8 slots of a kv head, shorter ones where that would leave less than 64 runs for the 8 XCDs
static inline void rp_blocks(RpArgs& a, int L, int T, int rows, int heads) {
    const int64_t n = rp_row_blocks(a, L, T, rows);
    int64_t main = n * heads;
    a.nrb = a.cu_q ? 0 : (L + rows - 1) / rows;
    a.slots = a.cu_q ? (int)std::min<int64_t>(n, RP_MAX_WGS) : 0;
    a.slot_group = 1;
    if (a.cu_q) {
        a.slot_group = (int)std::max<int64_t>(1, std::min<int64_t>(8, n * a.kv_heads / 64));
        const int64_t pairs = (n + a.slot_group - 1) / a.slot_group * a.kv_heads;
        main = a.B ? (pairs + 7) / 8 * 8 * a.slot_group * (heads / a.kv_heads) : 0;
    }
    a.nmain = main > RP_MAX_WGS ? -1 : (int)main;
}
// partial sums of ds over equal rel, per head
static inline int64_t rp_partials(const RpArgs& a, int rows, int qsplit) { return a.cu_q && !a.B ? 0 : rp_row_blocks(a, a.Lk, a.Tk, rows) * qsplit; }
// dK / dV of shared kv heads: a workgroup walks the rows of all G query heads; where that leaves less than two workgroups a CU, `parts` of them take G / parts
// heads each and rp_join_kv_kernel adds their fp32 sums (3 x 1023 causal, 16 / 4 heads, D = 128: 150 -> 75 us with the join;
// at RP_PART_STEPS chunks a walk, 4 x 256 rows of 16 / 4 heads, 37 -> 23, below that there is little to share out).  Not for packed sequences, whose
// lengths the host does not know.
#define RP_PART_STEPS 16
static inline int rp_dkv_parts(const RpArgs& a, int kt, int qsplit) {
    const int G = a.heads / a.kv_heads;
    const int64_t n = (int64_t)((a.Lk + 64 * kt - 1) / (64 * kt)) * a.B * a.kv_heads * qsplit;
    if (G == 1 || n == 0 || a.cu_q || (int64_t)((a.Lq + 63) / 64) * G / qsplit < RP_PART_STEPS) return 1;
    int p = 1;
    while (p < G && (G % p || n * p < 512)) ++p;
    return p;
}
// dK / dV of few keys against many query rows: the walk is cut every RP_SPLIT_ROWS (forward + backward, 11 x 3949 rows x 5 keys: 148 -> 79 us).  Shapes alone decide.
#define RP_SPLIT_ROWS 1024
static inline int rp_qsplit(const RpArgs& a) { return !a.cu_q && a.Lk <= 128 && a.Lq > RP_SPLIT_ROWS ? (a.Lq + RP_SPLIT_ROWS - 1) / RP_SPLIT_ROWS : 1; }
// the rows of a kv head's query heads fit the 16 columns of one tile (shapes of a sequence alone: its bits must not follow the batch)
static inline bool rp_few(const RpArgs& a) {
    return !a.cu_q && (int64_t)(a.heads / a.kv_heads) * a.Lq <= 16;
}
// splits over the keys: few query rows against many keys (single tokens, a handful of rows against a cache), joined by rp_join_kernel.  A number of keys that
// the shapes alone decide: a sequence's sums do not depend on the batch around it.  (3 x 47 rows of 4 heads against 4545 keys, fp32: 449 -> 148 us; dQ is split
// alike, joined by rp_join_q_kernel: forward + backward of 4 x 86 rows x 6756 keys 192 -> 102 us.)
static inline int rp_split_keys(int Lq) { return Lq <= 16 ? 512 : 1024; }
static inline int rp_nsplit(int Lq, int Lk, bool packed) {
    return !packed && Lq <= 128 && Lk > rp_split_keys(Lq) ? (Lk + rp_split_keys(Lq) - 1) / rp_split_keys(Lq) : 1;
}
