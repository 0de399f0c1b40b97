// Attention under a learned relative position bias, backward (operator and notation: relpos.h).  The probabilities are recomputed from the saved
// log-sum-exp:  p = exp(s - lse), dp = dout . v, delta = dout . out, ds = p (dp - delta);
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i      dv_j = sum_i p_ij dout_i      dtable[b, h] = sum over rel in bucket b of ds
// Two kernels, neither with an atomic on a gradient: rp_dq_kernel owns query rows and walks the keys (dq, delta), rp_dkv_kernel owns keys and walks the
// query rows of every head of its group (dk, dv, the sums for dtable).  Seven products instead of the five of the formulas; results do not depend on
// any order of arrival.
// Bound by vector issue beside the products (0.55 .. 0.6 and 0.36 of the cycles; two waves a SIMD, which overlap them only in part), no LDS conflicts.  12 heads,
// D = 64, bf16, no mask: 32 x 512 dQ 73 us, dK / dV 99 us (88 without the table's gradient; table sums 5 + 5); 4 x 4096 407 and 527 us, 770 TFLOP/s of the
// executed products together.  256 x 64 53 and 66, fp32 4 x 1024 at D = 128 370 and 489.
//
// delta.  sum_j ds_ij = 0, so a bucket that holds most of a row's probability has for its gradient what is left of a cancellation; delta taken from the
// bf16 `out` is off by up to 2^-8 of it, the same way for every element of the row (1 % of dtable measured, 40 queries against 3 .. 1500 keys).  What the
// ds of a row sum to instead of 0 IS that error (sum_j p_ij = 1): rp_dq_kernel sums them in fp32 on its way and hands the mended delta on
// (fp32 alike, where p's own rounding is what it mends: dtable 7.3e-7 -> 6.4e-7 of its norm, 6 x 1180 at D = 128).  Its own dq
// feels the error only where a row's probability sits on a few keys (by 1 / sqrt of their number), beside the rounding of ds to bf16 for the product with k.
// Row blocks of at most RP_FINE keys, and sequences of at most RP_FINE / 2 rows (too few values for roundings to average out), have ds as two bf16 parts there:
// dq within 1.8e-3 of its norm instead of 2.5e-3, one more product of the three, on blocks whose time is latency.  (A copy of the whole walk, FINE, in a
// kernel of its own instance, MIXED: as a branch inside the chunk it cost D = 128 its registers, 4 x 2048 200 -> 467 us, beside the walk 239 us; as a second
// launch it took 30 us more of a causal 3 x 1023 at D = 128, this way 11.)
//
// dtable.  In the accumulator layout lane (g, i16) holds ds of query 4 g + r (register r) and key i16, so -rel = const + 4 g + r - i16.  Moving register r
// by r lanes inside its 16 (a DPP operand modifier of the add itself) puts equal rel into equal lanes: the 16 x 16 tiles of one block diagonal add
// up in one register per lane, the lanes that fall off the end belong to the next block diagonal's register.  7 adds per 4 elements, no LDS; the registers
// live on from chunk to chunk until no later tile reaches their rel, and each sum is STORED once into the wave's own LDS bins (with ds_add_f32 instead,
// four a chunk, the kernel took 141 us against 107 at 32 x 512: LDS float atomics).  Chunks beyond the span add into one register per side instead (one add per element).
#include "relpos.h"
#include "relpos_launch.h"

#define RP_FINE 128

template <int CTRL>
__device__ __forceinline__ float rp_dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// acc[k], acc[k + 1] += the sums over equal rel of one 16 x 16 tile (block diagonal k): lane (g, i) of acc[k] stands for rel 16 k + 4 g - i
__device__ __forceinline__ void rp_diag_add(f32x4 x, float& lo, float& hi) {
    lo += x[0];
    lo += rp_dpp<0x101>(x[1]); hi += rp_dpp<0x11f>(x[1]);          // row_shl 1 / row_shr 15
    lo += rp_dpp<0x102>(x[2]); hi += rp_dpp<0x11e>(x[2]);
    lo += rp_dpp<0x103>(x[3]); hi += rp_dpp<0x11d>(x[3]);
}


// Four complete block diagonals x0 .. x3 -> one register of 64 sums, lane (row, i) = rel 16 row - i.  A lane's g-row is 4 g further: each register is turned by
// 4 g lanes inside its rows of 16 (one LDS permute), what goes past the end is the next diagonal's (`past` carries x3's to the next chunk), then the four rows
// add up in three exchanges.
__device__ __forceinline__ void rp_swap32(float& x, float& y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    x = __uint_as_float(r[0]); y = __uint_as_float(r[1]);
}
__device__ __forceinline__ void rp_swap16(float& x, float& y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    x = __uint_as_float(r[0]); y = __uint_as_float(r[1]);
}
__device__ __forceinline__ float rp_join4(float x0, float x1, float x2, float x3, float& past, int l) {
    const int g = l >> 4, i = l & 15, from = ((l & 48) | ((i + 4 * g) & 15)) * 4;
    const bool wrap = i + 4 * g >= 16;
    auto turn = [&](float x) { return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(from, __builtin_bit_cast(int, x))); };
    const float y0 = turn(x0), y1 = turn(x1), y2 = turn(x2), y3 = turn(x3);
    float z0 = wrap ? past : y0, z1 = wrap ? y0 : y1, z2 = wrap ? y1 : y2, z3 = wrap ? y2 : y3;
    past = y3;
    rp_swap32(z0, z2); rp_swap32(z1, z3);
    float a = z0 + z2, b = z1 + z3;
    rp_swap16(a, b);
    return a + b;
}

// keys that the 128-row block of row q0 may see, in whole chunks (the same for either QT: a row's bits must not depend on the grid)
__device__ __forceinline__ bool rp_fine(const RpArgs& a, const RpSeq& sq, int q0) {
    return (rp_seen(a, sq, q0 / 128 * 128 + 128) + 63) / 64 * 64 <= RP_FINE || sq.qn <= RP_FINE / 2;
}

// MIXED: row blocks may be FINE, or the keys are split (an instance of its own: what only these need costs the plain one 5 % at 4 x 4096 by its registers)
template <typename T, int DT, int QT_, bool MIXED>
__global__ __launch_bounds__(256, 2) void rp_dq_kernel(RpArgs a) {
    typedef RpTile<T, DT> Ti;
    constexpr int NB = rp_nb<T, DT>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    uint64_t* words = reinterpret_cast<uint64_t*>(smem + NB * 2 * Ti::BYTES);     // after the buffers of K and V chunks: the mask's words, the table
    float* tab = reinterpret_cast<float*>(words + a.mask_words);
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4, i16 = l & 15;
    const int nmain = a.nmain;
    const int nsplit = MIXED ? a.nsplit : 1, split = nmain ? (int)blockIdx.x / nmain : nsplit;
    if (split >= nsplit) {
        const int lead = rp_clamp(a.cu_q[0], 0, a.Tq), end = rp_clamp(a.cu_q[a.B], lead, a.Tq);
        rp_zero_rows((T*)a.dq, a.sdq, a.heads, a.D, lead, end, a.Tq, blockIdx.x - nmain * nsplit, RP_TAIL_WGS, tid);
        return;
    }
    constexpr int BQ_ = 64 * QT_;
    int slot, rb, h, b;
    if (!a.cu_q) rp_place(blockIdx.x - split * nmain, a.nrb, a.B, a.heads, a.kv_heads, a.causal, rb, h, b);
    else if (!rp_slot(a, a.cu_q, a.Tq, BQ_, a.heads, blockIdx.x, a.causal, slot, rb, h, b)) return;
    const RpSeq sq = rp_seq(a, b);
    constexpr bool AHEAD = sizeof(T) == 2;
    if (rb * BQ_ >= sq.qn) return;
    RpTable table;
    table.start(a, 1, tid);
    RpStage<T, DT> rk, rv;
    rk.init(a.sk.st, a.D, w, l); rv.init(a.sv.st, a.D, w, l);
    RpKeys keys;
    keys.init(a, sq, b, l, words);
    if (keys.m || a.causal || sq.kn % 64 || a.D != DT * 16) // (something of a chunk is not fetched)
        for (int t = 0; t < 2 * NB; ++t) rp_clear_own<T, DT>(smem + t * Ti::BYTES, w, l);
    rp_cleared();
    if (keys.m) { keys.build(words, w); __syncthreads(); }
    const int hk = h / (a.heads / a.kv_heads);
    const T* kb = (const T*)a.k + b * a.sk.sb + (int64_t)sq.k0 * a.sk.st + hk * a.sk.sh;
    const T* vb = (const T*)a.v + b * a.sv.sb + (int64_t)sq.k0 * a.sv.st + hk * a.sv.sh;
    const float c2 = a.scale * RP_LOG2E;
    const int mid = a.span + RP_PAD, span = a.span;
    const bool causal = a.causal;
    const int64_t rows = a.cu_q ? (int64_t)a.heads * a.Tq : (int64_t)a.B * a.heads * a.Lq;
    bool first = true;

    auto block = [&](auto qt_, auto fine_, const int q0) __attribute__((always_inline)) {
        constexpr int QT = decltype(qt_)::value, BQ = 64 * QT;
        constexpr bool FINE = decltype(fine_)::value;
        const int qw = q0 + w * 16 * QT;
        int c_from = 0, c_end = keys.upto(rp_seen(a, sq, q0 + BQ));
        if (MIXED && nsplit > 1) { c_from = split * (a.split_keys / 64); c_end = min(c_end, c_from + a.split_keys / 64); }
        typename Ti::frag fq[QT][Ti::KB], fdo[QT][Ti::KB];
        float nl[QT], rsum[QT];                             // -lse in the exponent's units; sum of a row's ds (each of its four lanes: a quarter of the keys)
        f32x4 nd[QT];                                       // -delta, as what the product dout . v starts from
        f32x4 dq[QT][DT];
#pragma unroll
        for (int ct = 0; ct < QT; ++ct) {
            rsum[ct] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) dq[ct][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
        auto fetch = [&](int at, int buf, uint64_t bits) {
            rk.load(kb + (int64_t)at * 64 * a.sk.st, bits, smem + buf * 2 * Ti::BYTES, w, l);
            rv.load(vb + (int64_t)at * 64 * a.sv.st, bits, smem + buf * 2 * Ti::BYTES + Ti::BYTES, w, l);
        };
        uint64_t bits;
        int c = keys.seek(c_from, c_end, bits), buf = 0;
        if (!first) __syncthreads();                    // (nobody is left in the buffers)
        if (NB == 2 && c < c_end) fetch(c, 0, bits);    // on its way before anything else is waited for
        typename Ti::frag fo[QT][Ti::KB];
        float lse[QT];                              // a row outside, or one that saw no key: -inf, and nl = -inf gives p = 0
#pragma unroll
        for (int ct = 0; ct < QT; ++ct) {
            const int q = qw + ct * 16 + i16;
            const bool ok = q < sq.qn;
            const int64_t qt = (int64_t)(sq.q0 + q);
#pragma unroll
            for (int kk = 0; kk < Ti::KB; ++kk) {
                fq[ct][kk] = Ti::gfrag((const T*)a.q + b * a.sq.sb + qt * a.sq.st + h * a.sq.sh, kk, g, a.D, ok);
                fdo[ct][kk] = Ti::gfrag((const T*)a.dout + b * a.sdo.sb + qt * a.sdo.st + h * a.sdo.sh, kk, g, a.D, ok);
                fo[ct][kk] = Ti::gfrag((const T*)a.o + b * a.so.sb + qt * a.so.st + h * a.so.sh, kk, g, a.D, ok);
            }
            lse[ct] = ok ? a.lse[rp_row(a, sq, b, h, q)] : -INFINITY;
        }
        if (first) table.finish(a, tab, h);
#pragma unroll
        for (int ct = 0; ct < QT; ++ct) {
            float acc = 0.f;
#pragma unroll
            for (int kk = 0; kk < Ti::KB; ++kk) acc += Ti::dot(fdo[ct][kk], fo[ct][kk]);
            acc += __shfl_xor(acc, 16, 64);
            acc += __shfl_xor(acc, 32, 64);
            nd[ct] = (f32x4){-acc, -acc, -acc, -acc};
            nl[ct] = lse[ct] == -INFINITY ? -INFINITY : lse[ct] == INFINITY ? NAN : -lse[ct] * RP_LOG2E;
        }
        first = false;
        auto chunk = [&](const bool near, const bool edge, const char* tK, int rel0, uint64_t now) __attribute__((always_inline)) {
            const char* tV = tK + Ti::BYTES;
            const float fc = near ? 0.f : tab[rel0 > 0 ? 2 * mid : 0] * c2;
            float al[QT];
#pragma unroll
            for (int ct = 0; ct < QT; ++ct) al[ct] = nl[ct] + fc;
            const float* bt = tab + (rel0 + mid + 4 * g - i16);
#pragma unroll
            for (int kp = 0; kp < 64 / Ti::KSTEP; ++kp) {
                f32x4 s[QT][Ti::RPS], dp[QT][Ti::RPS], z[Ti::RPS + QT - 1];
                rp_bias(near, bt, kp * Ti::RPS + 1 - QT, 0.f, z);
#pragma unroll
                for (int kk = 0; kk < Ti::KB; ++kk)
#pragma unroll
                    for (int j = 0; j < Ti::RPS; ++j) {
                        const int f = kp * Ti::RPS + j;
                        const typename Ti::frag fk = Ti::rowf(tK, f * 16 + i16, kk, g), fv = Ti::rowf(tV, f * 16 + i16, kk, g);
#pragma unroll
                        for (int ct = 0; ct < QT; ++ct) {
                            s[ct][j] = Ti::mma(fk, fq[ct][kk], kk == 0 ? rp_start<T>(z[j - ct + QT - 1]) : s[ct][j]);
                            dp[ct][j] = Ti::mma(fv, fdo[ct][kk], kk == 0 ? nd[ct] : dp[ct][j]);
                        }
                    }
                if (sizeof(T) == 4)
#pragma unroll
                    for (int j = 0; j < Ti::RPS; ++j)
#pragma unroll
                        for (int ct = 0; ct < QT; ++ct) s[ct][j] += z[j - ct + QT - 1];
                if (edge) {
#pragma unroll
                    for (int j = 0; j < Ti::RPS; ++j) {
                        const int f = kp * Ti::RPS + j;
                        const uint32_t nib = (uint32_t)(now >> (f * 16 + 4 * g));
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int ct = 0; ct < QT; ++ct)
                                s[ct][j][r] = ((nib >> r) & 1) && !(causal && rel0 + 16 * (f - ct) + 4 * g + r - i16 > 0) ? s[ct][j][r] : -INFINITY;
                    }
                }
                typename Ti::frag fds[QT], ahead;           // K fragments are read one step ahead, the first under the exponentials (fp32 has no registers for it)
                if constexpr (AHEAD) { ahead = Ti::colf(tK, kp, 0, l); __builtin_amdgcn_sched_barrier(0); }
#pragma unroll
                for (int ct = 0; ct < QT; ++ct) {
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < Ti::RPS; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            dp[ct][j][r] *= __builtin_amdgcn_exp2f(fmaf(s[ct][j][r], c2, al[ct]));
                            sum += dp[ct][j][r];
                        }
                    rsum[ct] += sum;
                    fds[ct] = Ti::pf(dp[ct]);
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const typename Ti::frag fk = AHEAD ? ahead : Ti::colf(tK, kp, d, l);
                    if (AHEAD && d + 1 < DT) ahead = Ti::colf(tK, kp, d + 1, l);
#pragma unroll
                    for (int ct = 0; ct < QT; ++ct) dq[ct][d] = Ti::mma(fk, fds[ct], dq[ct][d]);
                }
                if constexpr (FINE) {                       // what the rounding of ds left behind, as a second part
#pragma unroll
                    for (int ct = 0; ct < QT; ++ct) { Ti::less(dp[ct], fds[ct]); fds[ct] = Ti::pf(dp[ct]); }
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const typename Ti::frag fk = Ti::colf(tK, kp, d, l);
#pragma unroll
                        for (int ct = 0; ct < QT; ++ct) dq[ct][d] = Ti::mma(fk, fds[ct], dq[ct][d]);
                    }
                }
            }
        };
        while (c < c_end) {
            if (NB == 1) { __syncthreads(); fetch(c, 0, bits); }
            rp_landed();                                // this chunk is there, nobody reads the buffer of the one before it any more
            const char* tK = smem + buf * 2 * Ti::BYTES;
            const int rel0 = c * 64 - (qw + sq.off);
            const uint64_t now = bits;
            c = keys.seek(c + 1, c_end, bits);
            buf ^= NB - 1;
            if (NB == 2 && c < c_end) fetch(c, buf, bits);
            if (qw >= sq.qn || (causal && rel0 - (16 * QT - 1) > 0)) continue;
            const bool near = rp_near<T>(rel0, qw, span);
            chunk(near, now != ~0ull || (causal && rel0 + 63 > 0), tK, rel0, now);
        }
#pragma unroll
        for (int ct = 0; ct < QT; ++ct) {
            rsum[ct] += __shfl_xor(rsum[ct], 16, 64);
            rsum[ct] += __shfl_xor(rsum[ct], 32, 64);
        }
#pragma unroll
        for (int ct = 0; ct < QT; ++ct) {
            const int q = qw + ct * 16 + i16;
            if (q >= sq.qn) continue;
            const int64_t row = rp_row(a, sq, b, h, q);
            const bool blind = nl[ct] == -INFINITY;         // no key: no gradient, whatever dout holds there
            const float ndq = blind ? 0.f : nd[ct][0], rs = blind ? 0.f : rsum[ct];
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
            if (MIXED && nsplit > 1) {                      // rp_join_q_kernel adds them up
                float* op = a.part_q + (split * rows + row) * a.D;
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    if (d * 16 + g * 4 < a.D) *reinterpret_cast<f32x4*>(op + d * 16 + g * 4) = blind ? zero : dq[ct][d] * a.scale;
                if (g == 0) {
                    a.part_q[nsplit * rows * a.D + split * rows + row] = rs;
                    if (split == 0) { a.stat[row] = nl[ct]; a.stat[rows + row] = ndq; }
                }
                continue;
            }
            if (g == 0) { a.stat[row] = nl[ct]; a.stat[rows + row] = ndq - rs; }
            T* op = (T*)a.dq + b * a.sdq.sb + (int64_t)(sq.q0 + q) * a.sdq.st + h * a.sdq.sh;
#pragma unroll
            for (int d = 0; d < DT; ++d)
                if (d * 16 + g * 4 < a.D) Ti::st4(op + d * 16 + g * 4, blind ? zero : dq[ct][d] * a.scale);
        }
    };
    constexpr int FQ = DT <= 4 ? QT_ : 1;                   // (D > 64: 16 columns a wave, the second part needs the registers)
    if constexpr (MIXED && sizeof(T) == 2)
        if (rp_fine(a, sq, rb * BQ_)) {
            for (int q0 = rb * BQ_; q0 < min((rb + 1) * BQ_, sq.qn); q0 += 64 * FQ) block(std::integral_constant<int, FQ>(), std::true_type(), q0);
            return;
        }
    block(std::integral_constant<int, QT_>(), std::false_type(), rb * BQ_);
}

// CUT: the query heads of a group, or the query rows, are dealt over several workgroups (an instance of its own, as above)
template <typename T, int DT, int QT, bool CUT>
__global__ __launch_bounds__(256, DT * sizeof(T) * QT <= 16 ? 2 : 1) void rp_dkv_kernel(RpArgs a) {
    typedef RpTile<T, DT> Ti;
    constexpr int NB = rp_nb<T, DT>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int ND = 2 * (a.span + RP_PAD) + 1, mid = a.span + RP_PAD, span = a.span;
    float* rows = reinterpret_cast<float*>(smem + NB * 2 * Ti::BYTES);       // after the buffers of Q and dout chunks: the stat of their 64 rows
    float* tab = rows + NB * 128;                                // mirrored: entry x = bias of rel = -(x - mid), so that it ascends with the query
    float* bins = tab + ND;                                 // [4 waves][ND], mirrored like the table; only with part_d
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4, i16 = l & 15;
    const int parts = CUT ? a.parts : 1, qsplit = CUT ? a.qsplit : 1, nmain = a.nmain, split = nmain ? (int)blockIdx.x / nmain : qsplit;
    if (split >= qsplit) {
        const int lead = rp_clamp(a.cu_k[0], 0, a.Tk), end = rp_clamp(a.cu_k[a.B], lead, a.Tk);
        rp_zero_rows((T*)a.dk, a.sdk, a.kv_heads, a.D, lead, end, a.Tk, blockIdx.x - nmain * qsplit, RP_TAIL_WGS, tid);
        rp_zero_rows((T*)a.dv, a.sdv, a.kv_heads, a.D, lead, end, a.Tk, blockIdx.x - nmain * qsplit, RP_TAIL_WGS, tid);
        return;
    }
    constexpr int BK = 64 * QT;
    int slot = 0, rb, hp, b = 0;
    bool some = true;                                       // (packed: is there a row block of this number?)
    if (CUT || !a.cu_k) rp_place(blockIdx.x - split * nmain, a.nrb, a.B, a.kv_heads * parts, a.kv_heads, false, rb, hp, b);
    else {
        some = rp_slot(a, a.cu_k, a.Tk, BK, a.kv_heads, blockIdx.x, false, slot, rb, hp, b);
        if (slot >= a.slots) return;
    }
    const int hk = hp / parts, G = a.heads / a.kv_heads / parts, h0 = hp * G;       // this workgroup's query heads: h0 .. h0 + G - 1
    const RpSeq sq = rp_seq(a, b);
    const float c2 = a.scale * RP_LOG2E;
    const bool causal = a.causal;
    const int rows_k = a.cu_k ? sq.kn : a.Lk;               // padded: rows past k_lens are gradients of zero, and written
    const int64_t part_h = (int64_t)(CUT || !a.cu_k ? a.B * a.nrb * qsplit : a.slots) * ND;        // one head's partials
    float* part = a.part_d ? a.part_d + h0 * part_h + (int64_t)(CUT || !a.cu_k ? (b * a.nrb + rb) * qsplit + split : slot) * ND : nullptr;     // of the first head
    if (!some || rb * BK >= rows_k) {
        if (part)
            for (int gi = 0; gi < G; ++gi)
                for (int x = tid; x < ND; x += 256) part[gi * part_h + x] = 0.f;
        return;
    }
    float* bw = bins + w * ND;
    RpTable table;
    table.start(a, -1, tid);
    RpStage<T, DT> rq, ro;
    rq.init(a.sq.st, a.D, w, l); ro.init(a.sdo.st, a.D, w, l);
    if (a.causal || sq.qn % 64 || a.D != DT * 16) {         // (something of a chunk is not fetched)
        for (int t = 0; t < 2 * NB; ++t) rp_clear_own<T, DT>(smem + t * Ti::BYTES, w, l);
        if (w == 0)
            for (int x = l; x < NB * 128; x += 64) rows[x] = 0.f;
    }
    rp_cleared();
    const int64_t all_rows = a.cu_q ? (int64_t)a.heads * a.Tq : (int64_t)a.B * a.heads * a.Lq;

    const int k0 = rb * BK, kw = k0 + w * 16 * QT;
    int c_first = 0, n_ch = (sq.qn + 63) / 64, r_first = 0;
    if (causal) {                                       // query rows before r_first see none of these keys, and nothing of them is used
        int kf = k0;
        if (a.key_mask) {
            const uint8_t* m = a.key_mask + (a.cu_k ? (int64_t)sq.k0 : (int64_t)b * a.mask_sb);
            uint64_t vis = 0;
            for (; kf < min(k0 + BK, sq.kn) && !(vis = __ballot(kf + l < sq.kn && m[kf + l] != 0)); kf += 64) {}
            kf += vis ? __builtin_ctzll(vis) : 0;
        }
        r_first = max(0, kf - sq.off);
        c_first = r_first / 64;
    }
    if (CUT && qsplit > 1) { c_first = max(c_first, split * (RP_SPLIT_ROWS / 64)); n_ch = min(n_ch, (split + 1) * (RP_SPLIT_ROWS / 64)); }
    const T *qb, *ob;
    const float* stat_h;
    auto fetch = [&](int c, int buf) {
        const uint64_t ok = rp_low_bits(sq.qn - c * 64) & ~rp_low_bits(r_first - c * 64);
        rq.load(qb + (int64_t)c * 64 * a.sq.st, ok, smem + buf * 2 * Ti::BYTES, w, l);
        ro.load(ob + (int64_t)c * 64 * a.sdo.st, ok, smem + buf * 2 * Ti::BYTES + Ti::BYTES, w, l);
        if (w == 0 && ((ok >> l) & 1)) {                // 64 rows' stat: 4 bytes a lane
            amdseg_glds4(stat_h + c * 64 + l, rows + buf * 128);
            amdseg_glds4(stat_h + all_rows + c * 64 + l, rows + buf * 128 + 64);
        }
    };
    auto head = [&](int gi) {                           // a head's first chunk, on its way before anything else is waited for
        const int h = h0 + gi;
        qb = (const T*)a.q + b * a.sq.sb + (int64_t)sq.q0 * a.sq.st + h * a.sq.sh;
        ob = (const T*)a.dout + b * a.sdo.sb + (int64_t)sq.q0 * a.sdo.st + h * a.sdo.sh;
        stat_h = a.stat + rp_row(a, sq, b, h, 0);
        if (NB == 2 && c_first < n_ch) fetch(c_first, 0);
    };
    head(0);
    bool seen[QT];
    bool any = false, all = true;
    typename Ti::frag fk[QT][Ti::KB], fv[QT][Ti::KB];
#pragma unroll
    for (int ct = 0; ct < QT; ++ct) {
        const int key = kw + ct * 16 + i16;
        const bool in = key < rp_seen(a, sq, sq.qn);
        const int64_t kt = (int64_t)(sq.k0 + key);
        seen[ct] = in && (!a.key_mask || a.key_mask[(a.cu_k ? (int64_t)sq.k0 : (int64_t)b * a.mask_sb) + key] != 0);
#pragma unroll
        for (int kk = 0; kk < Ti::KB; ++kk) {
            fk[ct][kk] = Ti::gfrag((const T*)a.k + b * a.sk.sb + kt * a.sk.st + hk * a.sk.sh, kk, g, a.D, in);
            fv[ct][kk] = Ti::gfrag((const T*)a.v + b * a.sv.sb + kt * a.sv.st + hk * a.sv.sh, kk, g, a.D, in);
        }
    }
#pragma unroll
    for (int ct = 0; ct < QT; ++ct) {
        any |= seen[ct];
        all &= seen[ct];
    }
    const bool wave_any = __any(any), wave_all = __all(all);
    if (!wave_all)                                      // what stands in hidden rows reaches no product
#pragma unroll
        for (int ct = 0; ct < QT; ++ct)
#pragma unroll
            for (int kk = 0; kk < Ti::KB; ++kk) {
                fk[ct][kk] = seen[ct] ? fk[ct][kk] : (typename Ti::frag){};
                fv[ct][kk] = seen[ct] ? fv[ct][kk] : (typename Ti::frag){};
            }
    if (!__syncthreads_or(any)) { n_ch = 0; asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }      // (the chunk under way lands before anybody leaves)
    f32x4 dk[QT][DT], dv[QT][DT];
#pragma unroll
    for (int ct = 0; ct < QT; ++ct)
#pragma unroll
        for (int d = 0; d < DT; ++d) { dk[ct][d] = (f32x4){0.f, 0.f, 0.f, 0.f}; dv[ct][d] = (f32x4){0.f, 0.f, 0.f, 0.f}; }
    for (int gi = 0; gi < G; ++gi) {
        if (gi) { __syncthreads(); head(gi); }          // (nobody is left in the buffers, the table, the bins)
        table.finish(a, tab, h0 + gi);
        if (part)
            for (int x = tid; x < 4 * ND; x += 256) bins[x] = 0.f;
        int buf = 0;
        f32x4 far_sum = {0.f, 0.f, 0.f, 0.f};           // one side at a time: the chunks come in the order of -rel
        auto commit = [&](int at) {
            const float t = wave_sum(far_sum[0] + far_sum[1] + far_sum[2] + far_sum[3]);
            if (l == 0) bw[at] += t;
            far_sum = (f32x4){0.f, 0.f, 0.f, 0.f};
        };
        int side = 0;                                   // -1: rel >= span summed so far, 1: rel <= -span
        float diag[4 + QT], past = 0.f;                 // block diagonals 1 - QT .. 4 of the chunk
#pragma unroll
        for (int k = 0; k < 4 + QT; ++k) diag[k] = 0.f;
        auto chunk = [&](const bool near, const bool edge, const char* tQ, const float* rowl, int rel0, int there) __attribute__((always_inline)) {
            const char* tO = tQ + Ti::BYTES;
            const float* rowd = rowl + 64;
            const float* bt = tab + (rel0 + mid + 4 * g - i16);
            const float far = near ? 0.f : tab[rel0 > 0 ? 2 * mid : 0];
#pragma unroll
            for (int kp = 0; kp < 64 / Ti::KSTEP; ++kp) {
                f32x4 s[QT][Ti::RPS], dp[QT][Ti::RPS], lr[Ti::RPS], dr[Ti::RPS], z[Ti::RPS + QT - 1];
                rp_bias(near, bt, kp * Ti::RPS + 1 - QT, far, z);
#pragma unroll
                for (int j = 0; j < Ti::RPS; ++j) {
                    const int f = kp * Ti::RPS + j;
                    lr[j] = *reinterpret_cast<const f32x4*>(rowl + f * 16 + g * 4);
                    dr[j] = *reinterpret_cast<const f32x4*>(rowd + f * 16 + g * 4);
                }
#pragma unroll
                for (int kk = 0; kk < Ti::KB; ++kk)
#pragma unroll
                    for (int j = 0; j < Ti::RPS; ++j) {
                        const int f = kp * Ti::RPS + j;
                        const typename Ti::frag fq = Ti::rowf(tQ, f * 16 + i16, kk, g), fo = Ti::rowf(tO, f * 16 + i16, kk, g);
#pragma unroll
                        for (int ct = 0; ct < QT; ++ct) {
                            s[ct][j] = Ti::mma(fq, fk[ct][kk], kk == 0 ? rp_start<T>(z[j - ct + QT - 1]) : s[ct][j]);
                            dp[ct][j] = Ti::mma(fo, fv[ct][kk], kk == 0 ? dr[j] : dp[ct][j]);
                        }
                    }
                if (sizeof(T) == 4)
#pragma unroll
                    for (int j = 0; j < Ti::RPS; ++j)
#pragma unroll
                        for (int ct = 0; ct < QT; ++ct) s[ct][j] += z[j - ct + QT - 1];
                if (edge) {                             // a hidden key's column, rel > 0 with `causal`, a row behind the sequence: p = 0
#pragma unroll
                    for (int j = 0; j < Ti::RPS; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int row = (kp * Ti::RPS + j) * 16 + 4 * g + r;
#pragma unroll
                            for (int ct = 0; ct < QT; ++ct)
                                s[ct][j][r] = seen[ct] && row < there && !(causal && rel0 + row - 16 * ct - i16 < 0) ? s[ct][j][r] : -INFINITY;
                        }
                }
                typename Ti::frag fp[QT], fds[QT];
                constexpr bool AHEAD = sizeof(T) == 2;  // column fragments one step ahead, as in rp_dq_kernel
                typename Ti::frag fo, fq;
                if constexpr (AHEAD) { fo = Ti::colf(tO, kp, 0, l); fq = Ti::colf(tQ, kp, 0, l); __builtin_amdgcn_sched_barrier(0); }
#pragma unroll
                for (int ct = 0; ct < QT; ++ct) {
#pragma unroll
                    for (int j = 0; j < Ti::RPS; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float p = __builtin_amdgcn_exp2f(fmaf(s[ct][j][r], c2, lr[j][r]));
                            s[ct][j][r] = p;
                            dp[ct][j][r] *= p;
                        }
                    fp[ct] = Ti::pf(s[ct]);
                    fds[ct] = Ti::pf(dp[ct]);
                }
                if (part) {
                    if (near) {
                        // tiles of one block diagonal first add up element by element
#pragma unroll
                        for (int k = 0; k < Ti::RPS + QT - 1; ++k) {
                            f32x4 x = {0.f, 0.f, 0.f, 0.f};
                            bool have = false;
#pragma unroll
                            for (int j = 0; j < Ti::RPS; ++j)
#pragma unroll
                                for (int ct = 0; ct < QT; ++ct)
                                    if (j - ct + QT - 1 == k) {
                                        if (have) {
#pragma unroll
                                            for (int r = 0; r < 4; ++r) x[r] += dp[ct][j][r];
                                        } else x = dp[ct][j];
                                        have = true;
                                    }
                            rp_diag_add(x, diag[kp * Ti::RPS + k], diag[kp * Ti::RPS + k + 1]);
                        }
                    } else {
#pragma unroll
                        for (int ct = 0; ct < QT; ++ct)
#pragma unroll
                            for (int j = 0; j < Ti::RPS; ++j) far_sum += dp[ct][j];
                    }
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const typename Ti::frag co = AHEAD ? fo : Ti::colf(tO, kp, d, l), cq = AHEAD ? fq : Ti::colf(tQ, kp, d, l);
                    if (AHEAD && d + 1 < DT) { fo = Ti::colf(tO, kp, d + 1, l); fq = Ti::colf(tQ, kp, d + 1, l); }
#pragma unroll
                    for (int ct = 0; ct < QT; ++ct) {
                        dv[ct][d] = Ti::mma(co, fp[ct], dv[ct][d]);
                        dk[ct][d] = Ti::mma(cq, fds[ct], dk[ct][d]);
                    }
                }
            }
        };
        for (int c = c_first; c < n_ch; ++c, buf ^= NB - 1) {
            if (NB == 1) { __syncthreads(); fetch(c, 0); }
            rp_landed();
            const char* tQ = smem + buf * 2 * Ti::BYTES;
            const float* rowl = rows + buf * 128;
            if (NB == 2 && c + 1 < n_ch) fetch(c + 1, buf ^ 1);
            const int rel0 = c * 64 + sq.off - kw;      // (query - key) of the tile's first row and the wave's first column
            if (!wave_any || (causal && rel0 + 63 < 0)) continue;
            const bool near = rel0 + 63 > -span && rel0 - (16 * QT - 1) < span;
            if (part && side < 0 && rel0 > 0) { commit(0); side = 0; }
            if (part && !near) side = rel0 > 0 ? 1 : -1;
            chunk(near, !wave_all || (causal && rel0 - (16 * QT - 1) < 0) || (c + 1) * 64 > sq.qn, tQ, rowl, rel0, sq.qn - c * 64);
            if (part && near) {
                float* bd = bw + (rel0 - 16 * (QT - 1) + mid + 16 * g - i16);
                *bd = rp_join4(diag[0], diag[1], diag[2], diag[3], past, l);
                // the upper ones go on into the next chunk, 64 rel further; after the last near chunk they are stored too (nothing beyond rel0 + 63)
#pragma unroll
                for (int k = 0; k < QT; ++k) diag[k] = diag[4 + k];
#pragma unroll
                for (int k = QT; k < 4 + QT; ++k) diag[k] = 0.f;
                if (c + 1 >= n_ch || rel0 + 64 - (16 * QT - 1) >= span) {
                    const float rest = rp_join4(diag[0], QT > 1 ? diag[1] : 0.f, 0.f, 0.f, past, l);
                    if (64 - 16 * (QT - 1) + 16 * g - i16 <= 63) bd[64] = rest;
                    past = 0.f;
#pragma unroll
                    for (int k = 0; k < QT; ++k) diag[k] = 0.f;
                }
            }
        }
        if (part) {
            if (c_first >= n_ch) __syncthreads();       // (the zeroed bins: no chunk's barrier came in between)
            if (side) commit(side < 0 ? 0 : ND - 1);
            __syncthreads();
            for (int x = tid; x < ND; x += 256) {
                const float t = (bins[x] + bins[ND + x]) + (bins[2 * ND + x] + bins[3 * ND + x]);
                part[gi * part_h + (ND - 1 - x)] = t;
            }
        }
    }
    // a hidden key's column is zero, whatever dout held
#pragma unroll
    for (int ct = 0; ct < QT; ++ct) {
        const int key = kw + ct * 16 + i16;
        if (key >= rows_k) continue;
        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
        if (CUT) {
            const int64_t rows_all = (int64_t)a.B * a.Lk, row = (int64_t)b * a.Lk + key;
            float* kp_ = a.part_kv + ((((hp - hk * parts) * qsplit + split) * rows_all + row) * a.kv_heads + hk) * a.D;
            float* vp_ = kp_ + parts * qsplit * rows_all * a.kv_heads * a.D;
#pragma unroll
            for (int d = 0; d < DT; ++d)
                if (d * 16 + g * 4 < a.D) {
                    *reinterpret_cast<f32x4*>(kp_ + d * 16 + g * 4) = seen[ct] ? dk[ct][d] * a.scale : z;
                    *reinterpret_cast<f32x4*>(vp_ + d * 16 + g * 4) = seen[ct] ? dv[ct][d] : z;
                }
            continue;
        }
        T* kp_ = (T*)a.dk + b * a.sdk.sb + (int64_t)(sq.k0 + key) * a.sdk.st + hk * a.sdk.sh;
        T* vp_ = (T*)a.dv + b * a.sdv.sb + (int64_t)(sq.k0 + key) * a.sdv.st + hk * a.sdv.sh;
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (d * 16 + g * 4 < a.D) {
                Ti::st4(kp_ + d * 16 + g * 4, seen[ct] ? dk[ct][d] * a.scale : z);
                Ti::st4(vp_ + d * 16 + g * 4, seen[ct] ? dv[ct][d] : z);
            }
    }
}

// dk, dv = the sums of the parts * qsplit workgroups of a kv head, in their order.  Bound by its bytes (4 parts of 3 x 1023 x 4 x 128: 50 MB read).
template <typename T>
__global__ __launch_bounds__(256) void rp_join_kv_kernel(RpArgs a) {
    const int64_t one = (int64_t)a.B * a.Lk * a.kv_heads * a.D, x = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (x >= one) return;
    const int width = a.kv_heads * a.D, which = blockIdx.y;
    const int64_t row = x / width;
    const int hk = (int)(x % width) / a.D, d = (int)(x % width) % a.D;
    const float* p = a.part_kv + which * a.parts * a.qsplit * one + x;
    f32x4 s = *reinterpret_cast<const f32x4*>(p);
    for (int i = 1; i < a.parts * a.qsplit; ++i) s += *reinterpret_cast<const f32x4*>(p + i * one);
    const RpTensor& st = which ? a.sdv : a.sdk;
    const int64_t b = row / a.Lk, r = row % a.Lk;
    RpTile<T, 2>::st4((T*)(which ? a.dv : a.dk) + b * st.sb + r * st.st + hk * st.sh + d, s);
}

// dq and the mended delta of the splits over the keys, in their order (padded form).  A launch's latency: few rows, a handful of splits
template <typename T>
__global__ __launch_bounds__(256) void rp_join_q_kernel(RpArgs a) {
    const int64_t rows = (int64_t)a.B * a.heads * a.Lq, x = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (x >= rows * a.D) return;
    const int64_t row = x / a.D;
    const int d = (int)(x % a.D);
    f32x4 s = *reinterpret_cast<const f32x4*>(a.part_q + x);
    for (int i = 1; i < a.nsplit; ++i) s += *reinterpret_cast<const f32x4*>(a.part_q + i * rows * a.D + x);
    const int64_t bh = row / a.Lq, q = row % a.Lq;
    RpTile<T, 2>::st4((T*)a.dq + bh / a.heads * a.sdq.sb + q * a.sdq.st + bh % a.heads * a.sdq.sh + d, s);
    if (d == 0) {
        float rho = 0.f;
        for (int i = 0; i < a.nsplit; ++i) rho += a.part_q[a.nsplit * rows * a.D + i * rows + row];
        a.stat[rows + row] -= rho;
    }
}

// dtable from the workgroups' sums, in a fixed order: one workgroup per (bucket, head) lists the places of rel that belong to its bucket, then adds those of
// every partial.  Many partials (long batches): rp_sum_kernel first brings them down to one per head -- 64 places a workgroup, 16 interleaved groups.
__global__ __launch_bounds__(1024) void rp_sum_kernel(const float* part, float* sums, int64_t wgs, int nd) {
    __shared__ float red[16][64];
    const int x = blockIdx.x * 64 + (threadIdx.x & 63), y = threadIdx.x >> 6, h = blockIdx.y;
    float s = 0.f;
    if (x < nd) {
        const float* p = part + (h * wgs + y) * nd + x;
        int64_t i = y;
        for (; i + 48 < wgs; i += 64, p += (int64_t)64 * nd) {
            const float v0 = p[0], v1 = p[(int64_t)16 * nd], v2 = p[(int64_t)32 * nd], v3 = p[(int64_t)48 * nd];
            s += (v0 + v1) + (v2 + v3);
        }
        for (; i < wgs; i += 16, p += (int64_t)16 * nd) s += *p;
    }
    red[y][threadIdx.x & 63] = s;
    __syncthreads();
    if (y == 0 && x < nd) {
#pragma unroll
        for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x];
        sums[(int64_t)h * nd + x] = s;
    }
}
__global__ __launch_bounds__(256) void rp_bucket_kernel(const float* part, int wgs, const int* map, int span, int pad, int buckets, int heads, void* dtable,
                                                        int bf16) {
    __shared__ int list[2 * (RP_MAX_SPAN + RP_PAD) + 1];
    __shared__ int count[4];
    __shared__ float red[4];
    const int bk = blockIdx.x, h = blockIdx.y, nd = 2 * (span + pad) + 1, tid = threadIdx.x, w = tid >> 6, l = tid & 63;
    int len = 0;
    for (int x0 = 0; x0 < nd; x0 += 256) {
        const int x = x0 + tid;
        const bool mine = x < nd && rp_clamp(map[rp_clamp(x - span - pad, -span, span) + span], 0, buckets - 1) == bk;
        const uint64_t vote = __ballot(mine);
        if (l == 0) count[w] = __popcll(vote);
        __syncthreads();
        int at = len + __popcll(vote & ((1ull << l) - 1));
        for (int i = 0; i < w; ++i) at += count[i];
        if (mine) list[at] = x;
        len += count[0] + count[1] + count[2] + count[3];
        __syncthreads();
    }
    float s = 0.f;
    const float* p = part + (int64_t)h * wgs * nd;
    if (len > 0) {
        const int n = wgs * len;                            // (wgs <= 64)
        int i = tid / len, k = tid % len;
        const int di = 256 / len, dk = 256 % len;
#pragma unroll 4
        for (int x = tid; x < n; x += 256) {
            s += p[(int64_t)i * nd + list[k]];
            i += di; k += dk;
            if (k >= len) { k -= len; ++i; }
        }
    }
    s = wave_sum(s);
    if (l == 0) red[w] = s;
    __syncthreads();
    if (tid == 0) {
        s = (red[0] + red[1]) + (red[2] + red[3]);
        if (bf16) ((bf16_t*)dtable)[(int64_t)bk * heads + h] = f2bf(s);
        else ((float*)dtable)[(int64_t)bk * heads + h] = s;
    }
}
int amdseg_relpos_sums_impl(const float* part, float* sums, int64_t wgs, const int* map, int span, int pad, int buckets, int heads, void* dtable, int bf16,
                            hipStream_t s) {
    const int nd = 2 * (span + pad) + 1;
    const bool few = wgs <= 64;
    if (!few) {
        hipLaunchKernelGGL(rp_sum_kernel, dim3((nd + 63) / 64, heads), dim3(1024), 0, s, part, sums, wgs, nd);
        const int rc = amdseg_launch_status();
        if (rc) return rc;
    }
    hipLaunchKernelGGL(rp_bucket_kernel, dim3(buckets, heads), dim3(256), 0, s, few ? part : sums, few ? (int)wgs : 1, map, span, pad, buckets, heads, dtable, bf16);
    return amdseg_launch_status();
}

template <typename T, int DT, int QT, bool MIXED>
static int rp_dq_one(const RpArgs& a, int64_t n, int lds, hipStream_t s) {
    const int rc = rp_allow_lds((const void*)rp_dq_kernel<T, DT, QT, MIXED>, lds);
    if (rc) return rc;
    hipLaunchKernelGGL((rp_dq_kernel<T, DT, QT, MIXED>), dim3((unsigned)n), dim3(256), lds, s, a);
    return 0;
}
template <typename T, int DT, int QT>
static int rp_dkv_one(const RpArgs& a, int64_t n, int lds, hipStream_t s) {
    const bool cut = a.parts * a.qsplit > 1;
    const int rc = rp_allow_lds(cut ? (const void*)rp_dkv_kernel<T, DT, QT, true> : (const void*)rp_dkv_kernel<T, DT, QT, false>, lds);
    if (rc) return rc;
    if (cut) hipLaunchKernelGGL((rp_dkv_kernel<T, DT, QT, true>), dim3((unsigned)n), dim3(256), lds, s, a);
    else hipLaunchKernelGGL((rp_dkv_kernel<T, DT, QT, false>), dim3((unsigned)n), dim3(256), lds, s, a);
    return 0;
}
template <typename T, int DT>
static int rp_bwd_launch(RpArgs a, int dtype, void* dtable, float* sums, hipStream_t s) {
    const int ND = 2 * (a.span + RP_PAD) + 1;
    const int tail = a.zero_tail ? RP_TAIL_WGS : 0;
    a.mask_words = rp_mask_bytes(a) / 8;
    const int qt = rp_dq_qt(a, dtype), kt = rp_dkv_qt(a, dtype);
    rp_blocks(a, a.Lq, a.Tq, 64 * qt, a.heads);
    const int64_t n = (int64_t)a.nmain * a.nsplit + tail;
    if (a.nmain < 0 || n > RP_MAX_WGS) return AMDSEG_ERR_SHAPE;
    const int lds = 2 * rp_nb<T, DT> * RpTile<T, DT>::BYTES + a.mask_words * 8 + ND * 4;
    int rc = 0;
    if (n > 0) {
        if (sizeof(T) == 4) rc = a.nsplit > 1 ? rp_dq_one<T, DT, 1, true>(a, n, lds, s) : rp_dq_one<T, DT, 1, false>(a, n, lds, s);
        else if constexpr (sizeof(T) == 2) {                // can any row block be FINE?  Packed and ragged lengths are on the device
            const bool mixed = a.causal || a.cu_q || a.k_lens || a.Lk <= RP_FINE || a.Lq <= RP_FINE / 2 || a.nsplit > 1;
            if (mixed) rc = qt == 1 ? rp_dq_one<T, DT, 1, true>(a, n, lds, s) : rp_dq_one<T, DT, 2, true>(a, n, lds, s);
            else rc = qt == 1 ? rp_dq_one<T, DT, 1, false>(a, n, lds, s) : rp_dq_one<T, DT, 2, false>(a, n, lds, s);
        }
        if (rc) return rc;
    }
    if ((rc = amdseg_launch_status())) return rc;
    if (a.nsplit > 1 && n > 0) {
        const int64_t vecs = (int64_t)a.B * a.heads * a.Lq * (a.D / 4);
        if ((vecs + 255) / 256 > RP_MAX_WGS) return AMDSEG_ERR_SHAPE;
        hipLaunchKernelGGL(rp_join_q_kernel<T>, dim3((unsigned)((vecs + 255) / 256)), dim3(256), 0, s, a);
        if ((rc = amdseg_launch_status())) return rc;
    }
    a.qsplit = rp_qsplit(a);
    a.parts = rp_dkv_parts(a, kt, a.qsplit);
    rp_blocks(a, a.Lk, a.Tk, 64 * kt, a.kv_heads * a.parts);
    const int64_t m = (int64_t)a.nmain * a.qsplit + tail;
    if (a.nmain < 0 || m > RP_MAX_WGS) return AMDSEG_ERR_SHAPE;
    const int lds2 = rp_nb<T, DT> * (2 * RpTile<T, DT>::BYTES + 512) + ND * 4 * (a.part_d ? 5 : 1);
    if (m == 0) {
    } else if (sizeof(T) == 4 || DT > 4 || kt == 1) {
        rc = rp_dkv_one<T, DT, 1>(a, m, lds2, s);
    } else if constexpr (sizeof(T) == 2 && DT <= 4) {
        rc = rp_dkv_one<T, DT, 2>(a, m, lds2, s);
    }
    if (rc || (rc = amdseg_launch_status())) return rc;
    if (a.parts * a.qsplit > 1 && m > 0) {
        const int64_t vecs = (int64_t)a.B * a.Lk * a.kv_heads * (a.D / 4);
        if ((vecs + 255) / 256 > RP_MAX_WGS) return AMDSEG_ERR_SHAPE;
        hipLaunchKernelGGL(rp_join_kv_kernel<T>, dim3((unsigned)((vecs + 255) / 256), 2), dim3(256), 0, s, a);
        if ((rc = amdseg_launch_status())) return rc;
    }
    if (!a.part_d) return 0;
    return amdseg_relpos_sums_impl(a.part_d, sums, rp_partials(a, 64 * kt, a.qsplit), a.map, a.span, RP_PAD, a.buckets, a.heads, dtable, a.table_bf16, s);
}
template <typename T>
static int rp_bwd_d(const RpArgs& a, int dtype, void* dtable, float* sums, hipStream_t s) {
    return a.D <= 32 ? rp_bwd_launch<T, 2>(a, dtype, dtable, sums, s) : a.D <= 64 ? rp_bwd_launch<T, 4>(a, dtype, dtable, sums, s)
                                                                              : a.D <= 96 ? rp_bwd_launch<T, 6>(a, dtype, dtable, sums, s) : rp_bwd_launch<T, 8>(a, dtype, dtable, sums, s);
}
int amdseg_relpos_bwd_impl(const RpArgs& a, int dtype, void* dtable, float* sums, hipStream_t s) {
    return dtype == 1 ? rp_bwd_d<float>(a, dtype, dtable, sums, s) : rp_bwd_d<bf16_t>(a, dtype, dtable, sums, s);
}
