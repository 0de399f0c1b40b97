// Shared by the kernels of attention under a learned relative position bias (relpos_fwd.hip, relpos_bwd.hip): arguments, [64 rows] LDS tiles of both
// element types, fragment products, key visibility, the bias table of a workgroup.
//
//   s_ij = scale q_i . k_j + table[map[clamp(rel, -span, span) + span], h],   rel = j - (i + off)
//
// The bias depends on (i, j) through rel alone, so it is no [Lq, Lk] operand but a vector of 2 span + 1 floats per head.  A workgroup writes it into LDS
// once, extended by RP_PAD copies of the end values on both sides: a 64-row tile that touches |rel| < span then indexes without clamping, and a tile
// wholly beyond one end (almost all of a long sequence) starts from a constant and costs nothing.  It is kept divided by `scale`: MFMA accumulators START from
// it (fp32: it is added behind the products, rp_start) and scale * log2 e multiplies the finished score inside the exponent's fma.
#pragma once
#include <math.h>
#include <algorithm>
#include <type_traits>
#include "common.h"
#include "tile64.h"

#define RP_PAD 112              // 63 (tile rows) + 32 (columns of a wave, or of rp_near's group) + 15 lanes of the gradient's diagonal registers
#define RP_MAX_SPAN 1024
#define RP_MAX_WGS ((1 << 24) - 1)   // a grid has less than 2^32 threads
#define RP_LOG2E 1.4426950408889634f
#define RP_LN2 0.6931471805599453f

struct RpTensor { int64_t sb, st, sh; };     // element strides: sequence, token, head (last dimension contiguous)

struct RpArgs {
    const void *q, *k, *v; void* out; float* lse;
    const void *o, *dout; void *dq, *dk, *dv;
    RpTensor sq, sk, sv, so, sdo, sdq, sdk, sdv;
    const int *cu_q, *cu_k, *k_lens; const uint8_t* key_mask; int64_t mask_sb;
    const int* map; const void* table; int table_bf16;
    int B, Lq, Lk, heads, kv_heads, D, Tq, Tk, span, buckets, causal, align_end, zero_tail;
    float scale;
    int nrb;                    // padded: row blocks of a sequence
    int slots, slot_group;      // packed: row blocks of the batch (rp_slot), how many of them in a row stream the same K / V
    int nmain;                  // workgroups of one split (the others zero rows outside every sequence)
    int mask_words;             // 8-byte words of the key mask in LDS
    int nsplit, split_keys;     // forward and dQ: splits over the keys, keys of one (a multiple of 64)
    float* part_o; float* part_ml;           // forward, nsplit > 1: [nsplit][rows][D] unnormalised sums, [nsplit][rows][2] maximum and sum
    float* stat;                // backward: what the dK / dV kernel needs of a row: -lse in the exponent's units [rows], -sum_j p_ij dp_ij [rows]
    float* part_q;              // backward, nsplit > 1: [nsplit][rows][D] sums of dq, then [nsplit][rows] sums of ds
    int parts, qsplit;          // backward: workgroups that share a kv head's query heads, and its query rows, in the dK / dV kernel
    float* part_kv;             // backward, parts * qsplit > 1: [dk, dv][parts * qsplit][rows of k][kv_heads][D]
    float* part_d;              // backward: [heads][B * nrb * qsplit, or slots][2 (span + RP_PAD) + 1] sums of ds over equal rel, or NULL
};

// one sequence: where its rows start and how many there are.  The values of cu_q / cu_k / k_lens come from device memory that the host has not seen:
// they are clamped to the buffers here, so a wrong one gives wrong rows but no access outside.
struct RpSeq { int q0, qn, k0, kn, off; };
__device__ __forceinline__ int rp_clamp(int x, int lo, int hi) { return min(max(x, lo), hi); }
__device__ __forceinline__ RpSeq rp_seq(const RpArgs& a, int b) {
    RpSeq s;
    if (a.cu_q) {
        s.q0 = rp_clamp(a.cu_q[b], 0, a.Tq); s.qn = rp_clamp(a.cu_q[b + 1], s.q0, a.Tq) - s.q0;
        s.k0 = rp_clamp(a.cu_k[b], 0, a.Tk); s.kn = rp_clamp(a.cu_k[b + 1], s.k0, a.Tk) - s.k0;
    } else {
        s.q0 = 0; s.qn = a.Lq; s.k0 = 0;
        s.kn = a.k_lens ? rp_clamp(a.k_lens[b], 0, a.Lk) : a.Lk;
    }
    s.off = a.align_end ? s.kn - s.qn : 0;
    return s;
}
// the first `n` keys of a sequence are all that its query rows before `rows` may see
__device__ __forceinline__ int rp_seen(const RpArgs& a, const RpSeq& s, int rows) { return a.causal ? rp_clamp(min(rows, s.qn) + s.off, 0, s.kn) : s.kn; }
// index of (sequence b, head h, row i) in lse / delta
__device__ __forceinline__ int64_t rp_row(const RpArgs& a, const RpSeq& s, int b, int h, int i) {
    return a.cu_q ? (int64_t)h * a.Tq + s.q0 + i : ((int64_t)b * a.heads + h) * a.Lq + i;
}

// workgroup id -> (row block, head, sequence).  The row blocks (and the heads of a group) that stream the same K / V go to ONE XCD (ids are dealt round
// robin over the 8), so that its L2 fetches them once.  With a number of (sequence, kv head) pairs that is no multiple of 8 the row block is the slowest index:
// were it the fastest, a number of row blocks that IS a multiple of 8 would give one XCD all the long rows of a causal mask, or of ragged lengths (causal,
// 5 x 2048 at 12 heads: forward 107 -> 56 us, dq 128 -> 79, dk / dv 171 -> 108).
// `last_first`: row blocks from the last one down (under a causal mask the last has the most keys, and what is started last should be short).
__device__ __forceinline__ void rp_place(int id, int nrb, int B, int heads, int kv_heads, bool last_first, int& rb, int& h, int& b) {
    const int pairs = B * kv_heads, G = heads / kv_heads;
    int pair, gi;
    if ((pairs & 7) == 0) {
        const int t = id >> 3, rest = t % (nrb * G);
        pair = (t / (nrb * G)) * 8 + (id & 7);
        gi = rest / nrb; rb = rest % nrb;
    } else {
        const int rest = id % (pairs * G);
        rb = id / (pairs * G);
        pair = rest % pairs; gi = rest / pairs;
    }
    if (last_first) rb = nrb - 1 - rb;
    b = pair / kv_heads;
    h = (pair % kv_heads) * G + gi;
}

// The same for a packed batch, whose lengths the host does not know.  Row blocks of `rows` rows are numbered through (slots), T / rows + B numbers at most: grid
// and partial sums grow with the tokens, not with sequences times the longest.  Up to 64 sequences: one behind the other by a scan over their lengths, so that the
// numbers without a block come last (64 x 60 tokens: 9.2 us forward, 14 with a third of the workgroups empty in between).  More: sequence b's start at cu[b] / rows + b
// -- floor(y / rows) - floor(x / rows) + 1 >= ceil((y - x) / rows), so they fit -- and 64 candidates a step are looked at.  Every wave finds its sequence for
// itself.  Runs of `slot_group` slots of one kv head (mostly of one sequence) go to one XCD.
// -> false: no row block of this number (or none at all: slot >= a.slots)
__device__ __forceinline__ bool rp_slot(const RpArgs& a, const int* cu, int T, int rows, int heads, int id, bool last_first, int& slot, int& rb, int& h, int& b) {
    const int G = heads / a.kv_heads, sg = a.slot_group, t = id >> 3, rest = t % (sg * G), pair = t / (sg * G) * 8 + (id & 7);
    slot = pair / a.kv_heads * sg + rest % sg;
    h = pair % a.kv_heads * G + rest / sg;
    if (slot >= a.slots) return false;
    const int lane = threadIdx.x & 63;
    if (a.B <= 64) {
        const int from = rp_clamp(cu[min(lane, a.B)], 0, T), to = rp_clamp(cu[min(lane + 1, a.B)], from, T), n = lane < a.B ? (to - from + rows - 1) / rows : 0;
        int end = n;                                        // blocks of the sequences up to this lane's
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int x = __shfl_up(end, o, 64); end += lane >= o ? x : 0; }
        const int at = last_first ? __shfl(end, 63, 64) - 1 - slot : slot;
        const uint64_t vote = __ballot(end - n <= at && at < end);
        if (vote == 0) return false;
        b = __builtin_ctzll(vote);
        rb = __builtin_amdgcn_readlane(at - (end - n), b);
        return true;
    }
    const int at = last_first ? a.slots - 1 - slot : slot;
    int lo = 0, n = a.B;
    while (true) {
        const int step = (n + 63) / 64, x = lo + lane * step;
        const uint64_t vote = __ballot(lane * step < n && rp_clamp(cu[min(x, a.B)], 0, T) / rows + x <= at);
        if (vote == 0) return false;                        // in front of the first sequence
        const int k = __popcll(vote) - 1;
        lo += k * step;
        if (step == 1) break;
        n = min(step, n - k * step);
    }
    b = lo;
    rb = at - (rp_clamp(cu[b], 0, T) / rows + b);
    return rb >= 0;
}

// ------------------------------------------------------------------------------------------------ tiles and products
// RpTile<T, DT>: [64 rows][DT * 16 columns] in LDS.  A row fragment is the operand whose contraction runs along the columns (K of S^T = K Q^T), a
// column fragment the one whose contraction runs along the rows (V^T of O^T = V^T P^T).  PF(): accumulator registers of the score tiles as the other
// operand of that product -- the row order inside a contraction step is the accumulators' own, so the probabilities never move between lanes.
template <typename T, int DT> struct RpTile;
template <int DT> struct RpTile<bf16_t, DT> {
    typedef bf16x8 frag;
    static constexpr int BYTES = ((DT + 3) / 4) * 8192, KB = DT / 2, EPU = 8, UNITS = DT * 2;   // units = 16 bytes of a row
    static constexpr int KSTEP = 32, RPS = 2;                                                   // rows of a contraction step, 16-row tiles of it
    // piece p of 1 KiB: which row and 16-byte unit lane l's slot holds
    static __device__ __forceinline__ void piece(int p, int l, int& row, int& c) { row = (p & 7) * 8 + (l >> 3); c = (p >> 3) * 8 + ((l & 7) ^ swz(row)); }
    static __device__ __forceinline__ frag rowf(const char* t, int row, int kb, int g) { return at_frag(t + (kb >> 1) * 8192, row, (kb & 1) * 4 + g); }
    static __device__ __forceinline__ frag colf(const char* t, int step, int dt, int l) {
        const int g = l >> 4;
        return at_frag_tr(t + (dt >> 2) * 8192, step * 32 + g * 4, step * 32 + 16 + g * 4, (dt & 3) * 16, l);
    }
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ frag pf(const f32x4* s) {
        const uint4 u = make_uint4(pack2bf(s[0][0], s[0][1]), pack2bf(s[0][2], s[0][3]), pack2bf(s[1][0], s[1][1]), pack2bf(s[1][2], s[1][3]));
        return __builtin_bit_cast(frag, u);
    }
    // x - what pf() kept of x
    static __device__ __forceinline__ void less(f32x4* x, frag f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] -= bf2f((bf16_t)f[e]);
    }
    // the columns kb * 32 + g * 8 .. + 7 of one row of a global tensor, zero beyond D
    static __device__ __forceinline__ frag gfrag(const bf16_t* row, int kb, int g, int D, bool ok) {
        frag f = {0, 0, 0, 0, 0, 0, 0, 0};
        if (ok && kb * 32 + g * 8 < D) f = *reinterpret_cast<const frag*>(row + kb * 32 + g * 8);
        return f;
    }
    static __device__ __forceinline__ float dot(frag a, frag b) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s += bf2f((bf16_t)a[e]) * bf2f((bf16_t)b[e]);
        return s;
    }
    static __device__ __forceinline__ void st4(bf16_t* p, f32x4 v) { *reinterpret_cast<uint2*>(p) = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3])); }
};
template <int DT> struct RpTile<float, DT> {
    typedef f32x4 frag;
    static constexpr int BYTES = 64 * DT * 64, KB = DT, EPU = 4, UNITS = DT * 4;
    static constexpr int KSTEP = 16, RPS = 1;
    static __device__ __forceinline__ void piece(int p, int l, int& row, int& c) { row = (p * 64 + l) / UNITS; c = ((p * 64 + l) % UNITS) ^ (row & 7); }
    static __device__ __forceinline__ frag rowf(const char* t, int row, int kb, int g) {
        return *reinterpret_cast<const frag*>(t + row * (DT * 64) + (((kb * 4 + g) ^ (row & 7)) << 4));
    }
    static __device__ __forceinline__ frag colf(const char* t, int step, int dt, int l) {
        const int g = l >> 4, i16 = l & 15;
        frag f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = step * 16 + g * 4 + r;
            f[r] = *reinterpret_cast<const float*>(t + row * (DT * 64) + (((dt * 4 + (i16 >> 2)) ^ (row & 7)) << 4) + (i16 & 3) * 4);
        }
        return f;
    }
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ frag pf(const f32x4* s) { return s[0]; }
    static __device__ __forceinline__ void less(f32x4* x, frag) { x[0] = (f32x4){0.f, 0.f, 0.f, 0.f}; }
    static __device__ __forceinline__ frag gfrag(const float* row, int kb, int g, int D, bool ok) {
        frag f = {0.f, 0.f, 0.f, 0.f};
        if (ok && kb * 16 + g * 4 < D) f = *reinterpret_cast<const frag*>(row + kb * 16 + g * 4);
        return f;
    }
    static __device__ __forceinline__ float dot(frag a, frag b) { return a[0] * b[0] + a[1] * b[1] + a[2] * b[2] + a[3] * b[3]; }
    static __device__ __forceinline__ void st4(float* p, f32x4 v) { *reinterpret_cast<f32x4*>(p) = v; }
};

// 64 lanes x 16 bytes from base + lane offset to LDS.  The base may come straight from v_readfirstlane: a vector instruction's SGPR result needs five wait
// states before a memory instruction reads it, and the compiler does not look for them inside an asm statement
__device__ __forceinline__ void rp_glds16(const void* uniform_base, uint32_t lane_byte_offset, uint32_t lds_wave_addr) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(lane_byte_offset), "s"(uniform_base), "{m0}"(lds_wave_addr) : "memory");
}

// chunk buffers: two (the next chunk lands under this one's products), one where two would leave a CU a single workgroup (fp32, D > 64: the other
// workgroup's products hide the wait).  A third one, two chunks of lead, measured no faster at any length: 32 x 512 backward 83 + 147 us against 77 + 135.
template <typename T, int DT> constexpr int rp_nb = DT * sizeof(T) >= 32 ? 1 : 2;

// 64 rows of a tensor global -> LDS by the DMA path, 1 KiB a wave and instruction, no register in between.  The swizzle sits on the global side (lane l
// fetches what its fixed LDS slot holds).  Rows whose bit is clear and columns from D on are not fetched: their places keep what they held -- the zeros of
// rp_clear_own or a visible row of an earlier chunk -- so what stands in hidden rows (infinities, NaN) reaches no product, and a probability of exactly 0 meets
// a finite number.  (A key that `causal` hides from a part of a workgroup's rows is fetched.)
template <typename T, int DT> struct RpStage {
    typedef RpTile<T, DT> Ti;
    static constexpr int N = Ti::BYTES / 4096;              // pieces of a wave
    uint32_t off[N];                                        // byte offset of this lane's 16 bytes from the chunk's first row; ~0: beyond D
    bool full;
    __device__ __forceinline__ void init(int64_t st, int D, int w, int l) {
        full = D == DT * 16;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            int row, c;
            Ti::piece(w * N + n, l, row, c);
            off[n] = c < Ti::UNITS && c * Ti::EPU < D ? (uint32_t)(row * st * (int64_t)sizeof(T) + c * 16) : ~0u;
        }
    }
    __device__ __forceinline__ void load(const T* base, uint64_t bits, char* tile, int w, int l) const {
        const uint32_t lds = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)LDS_PTR(char, tile)) + w * N * 1024;
        const uint64_t u = (uint64_t)base;
        // (readfirstlane returns a signed int: without the casts the low half's sign bit would run into the high half)
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)u), hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
        const void* ub = (const void*)(((uint64_t)hi << 32) | lo);
        if (bits == ~0ull && full && DT % 4 == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) rp_glds16(ub, off[n], lds + n * 1024);
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                int row, c;
                Ti::piece(w * N + n, l, row, c);
                if (((bits >> row) & 1) && off[n] != ~0u) rp_glds16(ub, off[n], lds + n * 1024);
            }
        }
    }
};
// zeros into the pieces that this wave's own RpStage::load fills, before its first one (no barrier: nobody else writes there)
template <typename T, int DT>
__device__ __forceinline__ void rp_clear_own(char* tile, int w, int l) {
    constexpr int N = RpStage<T, DT>::N;
#pragma unroll
    for (int n = 0; n < N; ++n) *reinterpret_cast<uint4*>(tile + (w * N + n) * 1024 + l * 16) = make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ void rp_cleared() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void rp_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); __syncthreads(); }

// has a wave's chunk some |rel| < span (its scores start from the table) or none (from 0, the constant joins in the exponent)?  The two round differently, so in
// bf16 the 32 rows around the wave's decide, whether it has 16 of them or all: a row's bits do not follow the tiles that a grid chooses.
// `rel0` = rel of the chunk's first key and the wave's first query, which is row `qw`; RP_PAD covers the reach of the group's other half
template <typename T>
__device__ __forceinline__ bool rp_near(int rel0, int qw, int span) {
    constexpr int G = sizeof(T) == 2 ? 32 : 16;
    const int first = rel0 + (qw & (G - 1));                // ... and the group's first query
    return first + 63 > -span && first - (G - 1) < span;
}

// the bias values of the score tiles whose block diagonal (row tile - column tile) is k0, k0 + 1, ...: lane (g, i16), register r = rel 16 k + 4 g + r - i16
// (or `far`, where the whole tile is beyond the span)
template <int N>
__device__ __forceinline__ void rp_bias(bool near, const float* bt, int k0, float far, f32x4 (&z)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] = (f32x4){far, far, far, far};
    if (near)
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) z[k][r] = bt[16 * (k0 + k) + r];
}
// what a score's accumulator starts from: the bias itself, or (fp32) zero, the bias added behind the products -- every partial sum carries a rounding of its
// own size, and the bias would be in all of them (6 x 1180 at D = 128: out 9.2e-7 of its norm that way, 7.2e-7
// this way, as near as it gets in fp32; the additions are hidden by the fp32 products)
template <typename T>
__device__ __forceinline__ f32x4 rp_start(f32x4 bias) { return sizeof(T) == 2 ? bias : (f32x4){0.f, 0.f, 0.f, 0.f}; }

__device__ __forceinline__ uint64_t rp_low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// visible keys of a 64-key chunk as a wave-uniform word.  A key mask is turned into words in LDS by the workgroup before its first chunk (the chunk loop
// then has no load of its own whose wait would drain the chunks under way); only chunks beyond RP_MASK_WORDS (or a packed batch's hint) are looked up as
// they come.  `kn`: the keys that may be seen at all, of the sequence or (upto) of the rows at hand.
#define RP_MASK_WORDS 1024
struct RpKeys {
    const uint8_t* m; const uint64_t* words; int kn, lane, nw;
    __device__ __forceinline__ void init(const RpArgs& a, const RpSeq& s, int b, int lane_, uint64_t* lds) {
        m = a.key_mask ? a.key_mask + (a.cu_k ? (int64_t)s.k0 : (int64_t)b * a.mask_sb) : nullptr;
        words = lds; kn = s.kn; lane = lane_; nw = a.mask_words;
    }
    __device__ __forceinline__ int upto(int n) { kn = n; return (n + 63) / 64; }       // -> chunks that hold them
    __device__ __forceinline__ uint64_t look(int c) const { const int key = c * 64 + lane; return __ballot(key < kn && m[key] != 0); }
    __device__ __forceinline__ void build(uint64_t* lds, int w) const {       // (only with a mask; a barrier follows)
        const int n = min((kn + 63) / 64, nw);
        for (int c = w; c < n; c += 16) {
            uint32_t v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) { const int key = (c + 4 * u) * 64 + lane; v[u] = key < kn ? m[key] : 0; }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint64_t x = __ballot(v[u] != 0);
                if (lane == 0 && c + 4 * u < n) lds[c + 4 * u] = x;
            }
        }
    }
    __device__ __forceinline__ uint64_t bits(int c) const {
        const uint64_t low = rp_low_bits(kn - c * 64);
        if (!m) return low;
        if (c >= nw) return look(c);
        const uint64_t x = words[c];
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)), lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x);
        return low & (((uint64_t)hi << 32) | lo);
    }
    // the next chunk from c on that holds a visible key
    __device__ __forceinline__ int seek(int c, int c_end, uint64_t& w) const {
        w = 0;
        while (c < c_end && (w = bits(c)) == 0) ++c;
        return c;
    }
};
static inline int rp_mask_bytes(const RpArgs& a) { return a.key_mask ? 8 * std::min((a.Lk + 63) / 64, RP_MASK_WORDS) : 0; }

// LDS floats [2 (span + RP_PAD) + 1]: entry x = bias of rel = sign * (x - span - RP_PAD), divided by the scale.  Two dependent loads an entry: the first goes
// out with everything else a workgroup begins with (start), the second with its rows (finish), so that a workgroup pays two latencies before its
// first product and not one per load -- of 55 us for 32 x 512 forward 20 were such waits.
__device__ __forceinline__ float rp_table(const RpArgs& a, int bk, int h) {
    const int64_t at = (int64_t)rp_clamp(bk, 0, a.buckets - 1) * a.heads + h;
    return a.table_bf16 ? bf2f(((const bf16_t*)a.table)[at]) : ((const float*)a.table)[at];
}
// A finite entry of any size as a score.  Beyond +-RP_HUGE it is brought in by a logarithm, which keeps the order of entries: twice as large is RP_DOUBLING more,
// and e^-128 is 0.  Taken as they stand the largest would overflow over the scale or times log2 e, and a row that sees nothing else would have no
// digits left: q . k vanishes beside 1e9, and exp2(s - lse) in backward is off by the rounding of lse (2^-24 of it; 2^-10 at most here).  Infinities stay.
#define RP_HUGE 16384.f
#define RP_DOUBLING 128.f
__device__ __forceinline__ float rp_entry(float t) {
    const float x = fabsf(t);
    return x > RP_HUGE && x < INFINITY ? copysignf(RP_HUGE + RP_DOUBLING * __builtin_amdgcn_logf(x * (1.f / RP_HUGE)), t) : t;
}
__device__ __forceinline__ float rp_entry(const RpArgs& a, int bk, int h) { return rp_entry(rp_table(a, bk, h)); }
struct RpTable {
    int bk[2], n, mid, sign, tid;
    __device__ __forceinline__ int map(const RpArgs& a, int x) const { return a.map[rp_clamp(sign * (x - mid), -a.span, a.span) + a.span]; }
    __device__ __forceinline__ void start(const RpArgs& a, int sign_, int tid_) {
        mid = a.span + RP_PAD; n = 2 * mid + 1; sign = sign_; tid = tid_;
#pragma unroll
        for (int u = 0; u < 2; ++u) bk[u] = tid + 256 * u < n ? map(a, tid + 256 * u) : 0;
    }
    __device__ __forceinline__ void finish(const RpArgs& a, float* tab, int h) const {
        const float inv = 1.0f / a.scale;
        float v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) v[u] = rp_entry(a, bk[u], h);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (tid + 256 * u < n) tab[tid + 256 * u] = v[u] * inv;
        for (int x = tid + 512; x < n; x += 256) tab[x] = rp_entry(a, map(a, x), h) * inv;
    }
};
// zero rows [0, lead) and [end, T) of a packed tensor: `which` of `nwg` workgroups
template <typename T>
__device__ __forceinline__ void rp_zero_rows(T* p, const RpTensor& s, int heads, int D, int lead, int end, int T_, int which, int nwg, int tid) {
    const int64_t per = (int64_t)heads * (D / 4), n = (int64_t)(lead + T_ - end) * per;
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    for (int64_t i = (int64_t)which * 256 + tid; i < n; i += (int64_t)nwg * 256) {
        int64_t row = i / per;
        const int64_t rest = i % per;
        if (row >= lead) row += end - lead;
        RpTile<T, 2>::st4(p + row * s.st + (rest / (D / 4)) * s.sh + (rest % (D / 4)) * 4, z);
    }
}
#define RP_TAIL_WGS 32
