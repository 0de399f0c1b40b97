// Attention under a learned relative position bias, forward (operator and notation: relpos.h).  The framework's other attention kernels
// (attention.hip) take one interleaved projection with head_dim 64, whole 64-token blocks and an additive key mask.
//
// One workgroup = 4 waves x QT * 16 query rows of one (sequence, head); the keys stream through LDS in chunks of 64 with an online softmax.  S^T = K Q^T
// keeps a query in a lane (its maximum and sum are lane scalars, the probabilities are the second operand of O^T += V^T P^T as they stand).
// Bound by vector issue around the exponential, not by the products: a score costs its fma, its quarter-rate exponential, its share of maximum, sum and
// conversion against 4 D / 256 matrix cycles.  12 heads, D = 64, bf16, no mask, both products of every pair
// counted: 32 x 512 55 us (470 TFLOP/s, a third of it prologues and stores of 1536 workgroups), 4 x 4096 323 us (640), 1 x 16384 1.0 ms (820).
#include "relpos.h"
#include "relpos_launch.h"

template <typename T, int DT, int QT>
__global__ __launch_bounds__(256, 2) void rp_fwd_kernel(RpArgs a) {
    typedef RpTile<T, DT> Ti;
    constexpr int NB = rp_nb<T, DT>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    uint64_t* words = reinterpret_cast<uint64_t*>(smem + NB * 2 * Ti::BYTES);     // after the buffers of K and V chunks: the mask's words, the table
    float* tab = reinterpret_cast<float*>(words + a.mask_words);
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4, i16 = l & 15;
    int id = blockIdx.x;
    const int nmain = a.nmain, split = nmain ? id / nmain : a.nsplit;
    if (split >= a.nsplit) {                                // the buffer rows outside every sequence
        const int lead = rp_clamp(a.cu_q[0], 0, a.Tq), end = rp_clamp(a.cu_q[a.B], lead, a.Tq), which = id - nmain * a.nsplit;
        rp_zero_rows((T*)a.out, a.so, a.heads, a.D, lead, end, a.Tq, which, RP_TAIL_WGS, tid);
        if (a.lse)
            for (int h = 0; h < a.heads; ++h)
                for (int r = which * 256 + tid; r < lead + a.Tq - end; r += RP_TAIL_WGS * 256)
                    a.lse[(int64_t)h * a.Tq + (r < lead ? r : r - lead + end)] = -INFINITY;
        return;
    }
    id -= split * nmain;
    constexpr int BQ = 64 * QT;
    int slot, rb, h, b;
    if (!a.cu_q) rp_place(id, a.nrb, a.B, a.heads, a.kv_heads, a.causal, rb, h, b);
    else if (!rp_slot(a, a.cu_q, a.Tq, BQ, a.heads, id, a.causal, slot, rb, h, b)) return;
    const RpSeq sq = rp_seq(a, b);
    if (rb * BQ >= sq.qn) return;
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
    const T* qbase = (const T*)a.q + b * a.sq.sb + (int64_t)sq.q0 * a.sq.st + h * a.sq.sh;
    const float c2 = a.scale * RP_LOG2E;
    const int mid = a.span + RP_PAD, span = a.span;
    const bool causal = a.causal;

    const int q0 = rb * BQ, qw = q0 + w * 16 * QT;
    int c = 0, c_end = keys.upto(rp_seen(a, sq, q0 + BQ));
    if (a.nsplit > 1) { c = split * (a.split_keys / 64); c_end = min(c_end, c + a.split_keys / 64); }
    auto fetch = [&](int at, int buf, uint64_t bits) {
        rk.load(kb + (int64_t)at * 64 * a.sk.st, bits, smem + buf * 2 * Ti::BYTES, w, l);
        rv.load(vb + (int64_t)at * 64 * a.sv.st, bits, smem + buf * 2 * Ti::BYTES + Ti::BYTES, w, l);
    };
    uint64_t bits;
    c = keys.seek(c, c_end, bits);
    int buf = 0;
    if (NB == 2 && c < c_end) fetch(c, 0, bits);        // on its way before anything else is waited for
    typename Ti::frag fq[QT][Ti::KB];
#pragma unroll
    for (int ct = 0; ct < QT; ++ct) {
        const int q = qw + ct * 16 + i16;
#pragma unroll
        for (int kk = 0; kk < Ti::KB; ++kk) fq[ct][kk] = Ti::gfrag(qbase + (int64_t)q * a.sq.st, kk, g, a.D, q < sq.qn);
    }
    table.finish(a, tab, h);
    f32x4 o[QT][DT];
    float m_run[QT], l_part[QT];
#pragma unroll
    for (int ct = 0; ct < QT; ++ct) {
        m_run[ct] = -INFINITY; l_part[ct] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[ct][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    // one chunk: `near` = some |rel| < span (scores start from the table; else from 0, and the constant joins in the exponent), `edge` = some (i, j) hidden
    auto chunk = [&](const bool near, const bool edge, const char* tK, int rel0, uint64_t now) __attribute__((always_inline)) {
        const char* tV = tK + Ti::BYTES;
        f32x4 s[QT][4], z[3 + QT];
        rp_bias(near, tab + (rel0 + mid + 4 * g - i16), 1 - QT, 0.f, z);
#pragma unroll
        for (int kk = 0; kk < Ti::KB; ++kk)
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const typename Ti::frag fk = Ti::rowf(tK, f * 16 + i16, kk, g);
#pragma unroll
                for (int ct = 0; ct < QT; ++ct) {
                    s[ct][f] = Ti::mma(fk, fq[ct][kk], kk == 0 ? rp_start<T>(z[f - ct + QT - 1]) : s[ct][f]);
                }
            }
        if (sizeof(T) == 4)
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int ct = 0; ct < QT; ++ct) s[ct][f] += z[f - ct + QT - 1];
        if (edge) {
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const uint32_t nib = (uint32_t)(now >> (f * 16 + 4 * g));
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int ct = 0; ct < QT; ++ct)
                        s[ct][f][r] = ((nib >> r) & 1) && !(causal && rel0 + 16 * (f - ct) + 4 * g + r - i16 > 0) ? s[ct][f][r] : -INFINITY;
            }
        }
        const float fc = near ? 0.f : tab[rel0 > 0 ? 2 * mid : 0] * c2;
        typename Ti::frag ahead = Ti::colf(tV, 0, 0, l);        // V fragments are read one step ahead: the first under the exponentials
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ct = 0; ct < QT; ++ct) {
            float mx = s[ct][0][0];
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[ct][f][r]);
            mx = fmaf(mx, c2, fc);
            if (__any(mx > m_run[ct])) {                // wave-uniform: some row's running maximum grows
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float m_new = fmaxf(m_run[ct], mx);
                const float al = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[ct] - m_new);
                m_run[ct] = m_new;
                l_part[ct] *= al;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[ct][d][r] *= al;
            }
            const float mu = fc - (m_run[ct] == -INFINITY ? 0.f : m_run[ct]);
            float sum = 0.f;
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(s[ct][f][r], c2, mu));
                    s[ct][f][r] = e;
                    sum += e;
                }
            l_part[ct] += sum;
        }
#pragma unroll
        for (int kp = 0; kp < 64 / Ti::KSTEP; ++kp) {
            typename Ti::frag fp[QT];
#pragma unroll
            for (int ct = 0; ct < QT; ++ct) fp[ct] = Ti::pf(&s[ct][kp * Ti::RPS]);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const typename Ti::frag fv = ahead;
                if (d + 1 < DT) ahead = Ti::colf(tV, kp, d + 1, l);
                else if (kp + 1 < 64 / Ti::KSTEP) ahead = Ti::colf(tV, kp + 1, 0, l);
#pragma unroll
                for (int ct = 0; ct < QT; ++ct) o[ct][d] = Ti::mma(fv, fp[ct], o[ct][d]);
            }
        }
    };
    while (c < c_end) {
        if (NB == 1) { __syncthreads(); fetch(c, 0, bits); }
        rp_landed();                                    // this chunk is there (and the table), nobody reads the buffer of the one before it any more
        const char* tK = smem + buf * 2 * Ti::BYTES;
        const int rel0 = c * 64 - (qw + sq.off);        // rel of the chunk's first key and the wave's first query
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
        const int q = qw + ct * 16 + i16;
        float ls = l_part[ct];
        ls += __shfl_xor(ls, 16, 64);
        ls += __shfl_xor(ls, 32, 64);
        if (q >= sq.qn) continue;
        const int64_t row = rp_row(a, sq, b, h, q);
        if (a.nsplit > 1) {
            const int64_t rows = a.cu_q ? (int64_t)a.heads * a.Tq : (int64_t)a.B * a.heads * a.Lq;
            float* po = a.part_o + (split * rows + row) * a.D;
#pragma unroll
            for (int d = 0; d < DT; ++d)
                if (d * 16 + g * 4 < a.D) *reinterpret_cast<f32x4*>(po + d * 16 + g * 4) = o[ct][d];
            if (g == 0) { a.part_ml[(split * rows + row) * 2] = m_run[ct]; a.part_ml[(split * rows + row) * 2 + 1] = ls; }
            continue;
        }
        const float inv = ls > 0.f ? 1.0f / ls : (ls == 0.f ? 0.f : ls);    // a row that saw no key: zero; NaN stays
        T* op = (T*)a.out + b * a.so.sb + (int64_t)(sq.q0 + q) * a.so.st + h * a.so.sh;
#pragma unroll
        for (int d = 0; d < DT; ++d)
            if (d * 16 + g * 4 < a.D) Ti::st4(op + d * 16 + g * 4, o[ct][d] * inv);
        if (a.lse && g == 0) a.lse[row] = ls == 0.f ? -INFINITY : (m_run[ct] + __builtin_amdgcn_logf(ls)) * RP_LN2;
    }
}

// The few-rows form: single tokens (or a handful) against a cache.  HBM-bound, so K and V are read once: the G query heads of a kv head and their Lq rows, at most
// 16 together, are the 16 columns of one tile.  A workgroup has one split of one (sequence, kv head); its four waves take the split's 64-key chunks in turn and
// need nothing from each other until the end: K goes straight into registers (its row fragments are 16 contiguous bytes), V through the wave's own LDS piece
// for the transposed read (one token of 16 sequences of 700 .. 4096 keys, 16 / 4 heads,
// D = 128: 88 MB in 25 us, 3.5 TB/s).  No bias table in LDS (every column has another head): only the chunks within the span of the rows look values up.
template <typename T, int DT>
__global__ __launch_bounds__(256, DT * sizeof(T) >= 32 ? 1 : 2) void rp_few_kernel(RpArgs a) {
    typedef RpTile<T, DT> Ti;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float ml[4][16][2];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4, i16 = l & 15;
    const int split = blockIdx.x, pair = blockIdx.z * gridDim.y + blockIdx.y, b = pair / a.kv_heads, hk = pair % a.kv_heads;
    if (b >= a.B) return;
    const int G = a.heads / a.kv_heads;
    const RpSeq sq = rp_seq(a, b);
    char* tV = smem + w * Ti::BYTES;
    const bool col_ok = i16 < G * a.Lq;
    const int qi = col_ok ? i16 / G : 0, h = hk * G + (col_ok ? i16 % G : 0), pos = qi + sq.off;
    RpKeys keys;
    keys.init(a, sq, b, l, nullptr);
    keys.nw = 0;                                            // (the mask as it comes: a wave sees two or three chunks of it)
    const bool causal = a.causal;
    int c_end = keys.upto(rp_seen(a, sq, a.Lq));
    const int c0 = split * (a.split_keys / 64);
    c_end = a.nsplit > 1 ? min(c_end, c0 + a.split_keys / 64) : c_end;
    typename Ti::frag fq[Ti::KB];
    {
        const T* qrow = (const T*)a.q + b * a.sq.sb + (int64_t)qi * a.sq.st + h * a.sq.sh;
#pragma unroll
        for (int kk = 0; kk < Ti::KB; ++kk) fq[kk] = Ti::gfrag(qrow, kk, g, a.D, col_ok);
    }
    const float c2 = a.scale * RP_LOG2E, farL = rp_entry(a, a.map[0], h) * RP_LOG2E, farR = rp_entry(a, a.map[2 * a.span], h) * RP_LOG2E;
    if (keys.m || keys.kn % 64 || a.D != DT * 16) {
#pragma unroll
        for (int n = 0; n < Ti::BYTES / 1024; ++n) *reinterpret_cast<uint4*>(tV + n * 1024 + l * 16) = make_uint4(0u, 0u, 0u, 0u);
        rp_cleared();
    }
    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_part = 0.f;
    for (int c = c0 + w; c < c_end; c += 4) {
        const uint64_t now = keys.bits(c);
        if (now == 0) continue;
        const T* kb = (const T*)a.k + b * a.sk.sb + (int64_t)c * 64 * a.sk.st + hk * a.sk.sh;
        const uint64_t va = (uint64_t)((const T*)a.v + b * a.sv.sb + (int64_t)c * 64 * a.sv.st + hk * a.sv.sh);
        typename Ti::frag fk[4][Ti::KB];
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int kk = 0; kk < Ti::KB; ++kk) fk[f][kk] = Ti::gfrag(kb + (int64_t)(f * 16 + i16) * a.sk.st, kk, g, a.D, (now >> (f * 16 + i16)) & 1);
        const void* vbase = (const void*)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(va >> 32)) << 32) |
                                          (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)va));
        const uint32_t lds = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)LDS_PTR(char, tV));
#pragma unroll
        for (int n = 0; n < Ti::BYTES / 1024; ++n) {
            int row, u;
            Ti::piece(n, l, row, u);
            if (((now >> row) & 1) && u < Ti::UNITS && u * Ti::EPU < a.D)
                rp_glds16(vbase, (uint32_t)row * (uint32_t)(a.sv.st * (int64_t)sizeof(T)) + u * 16, lds + n * 1024);
        }
        const int rel0 = c * 64 + 4 * g - pos;
        const bool near = c * 64 + 63 - sq.off > -a.span && c * 64 - (sq.off + a.Lq - 1) < a.span;
        f32x4 s[4], z[4];
        if (near) {
            const float inv = 1.0f / a.scale;
            int bk[4][4];
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int r = 0; r < 4; ++r) bk[f][r] = a.map[rp_clamp(rel0 + 16 * f + r, -a.span, a.span) + a.span];
            bool huge = false;
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int r = 0; r < 4; ++r) { z[f][r] = rp_table(a, bk[f][r], h); huge |= fabsf(z[f][r]) > RP_HUGE; }
            if (__any(huge))
#pragma unroll
                for (int f = 0; f < 4; ++f)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z[f][r] = rp_entry(z[f][r]);
#pragma unroll
            for (int f = 0; f < 4; ++f) z[f] *= inv;
        } else
#pragma unroll
            for (int f = 0; f < 4; ++f) z[f] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < Ti::KB; ++kk)
#pragma unroll
            for (int f = 0; f < 4; ++f) s[f] = Ti::mma(fk[f][kk], fq[kk], kk == 0 ? rp_start<T>(z[f]) : s[f]);
        if (sizeof(T) == 4)
#pragma unroll
            for (int f = 0; f < 4; ++f) s[f] += z[f];
        const float fc = near ? 0.f : c * 64 > sq.off ? farR : farL;
        if (now != ~0ull || causal)
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const uint32_t nib = (uint32_t)(now >> (f * 16 + 4 * g));
#pragma unroll
                for (int r = 0; r < 4; ++r) s[f][r] = ((nib >> r) & 1) && !(causal && rel0 + 16 * f + r > 0) ? s[f][r] : -INFINITY;
            }
        float mx = s[0][0];
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[f][r]);
        mx = fmaf(mx, c2, fc);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m_run, mx);
        const float al = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new), mu = fc - (m_new == -INFINITY ? 0.f : m_new);
        m_run = m_new;
        float sum = 0.f;
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[f][r], c2, mu));
                s[f][r] = e;
                sum += e;
            }
        l_part = l_part * al + sum;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[d][r] *= al;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int kp = 0; kp < 64 / Ti::KSTEP; ++kp) {
            const typename Ti::frag fp = Ti::pf(&s[kp * Ti::RPS]);
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = Ti::mma(Ti::colf(tV, kp, d, l), fp, o[d]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the piece has been read before the next chunk lands in it)
    }
    // the four waves' sums meet in LDS, each in its own piece: [16 columns][D]
    l_part += __shfl_xor(l_part, 16, 64);
    l_part += __shfl_xor(l_part, 32, 64);
    float* mine = reinterpret_cast<float*>(tV);
#pragma unroll
    for (int d = 0; d < DT; ++d)
        if (d * 16 + g * 4 < a.D) *reinterpret_cast<f32x4*>(mine + i16 * (DT * 16) + d * 16 + g * 4) = o[d];
    if (g == 0) { ml[w][i16][0] = m_run; ml[w][i16][1] = l_part; }
    __syncthreads();
    const int col = tid >> 4, d0 = (tid & 15) * 8;
    if (col >= G * a.Lq) return;
    float m = ml[0][col][0];
#pragma unroll
    for (int i = 1; i < 4; ++i) m = fmaxf(m, ml[i][col][0]);
    const float mu = m == -INFINITY ? 0.f : m;
    float ls = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float f = __builtin_amdgcn_exp2f(ml[i][col][0] - mu);
        ls += f * ml[i][col][1];
        if (d0 < a.D) {
            const float* p = reinterpret_cast<const float*>(smem + i * Ti::BYTES) + col * (DT * 16) + d0;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] += f * p[e];
        }
    }
    const int q = col / G, hh = hk * G + col % G;
    const int64_t row = rp_row(a, sq, b, hh, q);
    if (a.nsplit > 1) {
        const int64_t at = split * ((int64_t)a.B * a.heads * a.Lq) + row;
        if (d0 < a.D) {
            *reinterpret_cast<f32x4*>(a.part_o + at * a.D + d0) = (f32x4){x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(a.part_o + at * a.D + d0 + 4) = (f32x4){x[4], x[5], x[6], x[7]};
        }
        if (d0 == 0) { a.part_ml[at * 2] = m; a.part_ml[at * 2 + 1] = ls; }
        return;
    }
    const float inv = ls > 0.f ? 1.0f / ls : (ls == 0.f ? 0.f : ls);
    if (d0 < a.D) {
        T* op = (T*)a.out + b * a.so.sb + (int64_t)q * a.so.st + hh * a.so.sh + d0;
        Ti::st4(op, (f32x4){x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv});
        Ti::st4(op + 4, (f32x4){x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv});
    }
    if (a.lse && d0 == 0) a.lse[row] = ls == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(ls)) * RP_LN2;
}

// the splits of a row joined in their order: one wave per row, lane s first has split s's maximum and sum
template <typename T>
__global__ __launch_bounds__(256) void rp_join_kernel(RpArgs a) {
    const int l = threadIdx.x & 63;
    const int64_t rows = (int64_t)a.B * a.heads * a.Lq;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    float m = -INFINITY;
    for (int s = l; s < a.nsplit; s += 64) m = fmaxf(m, a.part_ml[(s * rows + row) * 2]);
    m = wave_max(m);
    const float mu = m == -INFINITY ? 0.f : m;
    float ls = 0.f, x0 = 0.f, x1 = 0.f;
    const int d = l * 2;
    const float* p = a.part_o + row * a.D + (d < a.D ? d : 0);
    for (int s0 = 0; s0 < a.nsplit; s0 += 64) {
        const int s = s0 + l;
        const float f = s < a.nsplit ? __builtin_amdgcn_exp2f(a.part_ml[(s * rows + row) * 2] - mu) : 0.f;
        ls += s < a.nsplit ? f * a.part_ml[(s * rows + row) * 2 + 1] : 0.f;
        const int n = min(64, a.nsplit - s0);
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const float fi = __shfl(f, i, 64);
            const float2 v = *reinterpret_cast<const float2*>(p + (s0 + i) * rows * a.D);
            x0 += fi * v.x; x1 += fi * v.y;
        }
    }
    ls = wave_sum(ls);
    const float inv = ls > 0.f ? 1.0f / ls : (ls == 0.f ? 0.f : ls);
    const int i = (int)(row % a.Lq), h = (int)(row / a.Lq % a.heads), b = (int)(row / a.Lq / a.heads);
    T* op = (T*)a.out + b * a.so.sb + (int64_t)i * a.so.st + h * a.so.sh;
    if (d < a.D) { Act<T>::st(op + d, x0 * inv); Act<T>::st(op + d + 1, x1 * inv); }
    if (a.lse && l == 0) a.lse[row] = ls == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(ls)) * RP_LN2;
}

template <typename T, int DT>
static int rp_few_launch(const RpArgs& a, hipStream_t s) {
    const int lds = 4 * RpTile<T, DT>::BYTES;
    const int rc = rp_allow_lds((const void*)rp_few_kernel<T, DT>, lds);
    if (rc) return rc;
    const int64_t pairs = (int64_t)a.B * a.kv_heads, y = std::min<int64_t>(pairs, 65535), z = (pairs + 65534) / 65535;
    if (z > 4096) return AMDSEG_ERR_SHAPE;                  // (pair numbers stay below 2^28)
    hipLaunchKernelGGL((rp_few_kernel<T, DT>), dim3(a.nsplit, (unsigned)y, (unsigned)z), dim3(256), lds, s, a);
    return amdseg_launch_status();
}
template <typename T>
static int rp_join_launch(const RpArgs& a, hipStream_t s) {
    if (a.nsplit > 1) {
        const int64_t rows = (int64_t)a.B * a.heads * a.Lq;
        if ((rows + 3) / 4 > RP_MAX_WGS) return AMDSEG_ERR_SHAPE;
        hipLaunchKernelGGL((rp_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
    }
    return amdseg_launch_status();
}

template <typename T, int DT, int QT>
static int rp_fwd_launch(const RpArgs& a, hipStream_t s) {
    const int lds = 2 * rp_nb<T, DT> * RpTile<T, DT>::BYTES + a.mask_words * 8 + (2 * (a.span + RP_PAD) + 1) * 4;
    const int rc = rp_allow_lds((const void*)rp_fwd_kernel<T, DT, QT>, lds);
    if (rc) return rc;
    const int64_t n = (int64_t)a.nmain * a.nsplit + (a.zero_tail ? RP_TAIL_WGS : 0);
    if (a.nmain < 0 || n > RP_MAX_WGS) return AMDSEG_ERR_SHAPE;
    if (n == 0) return 0;                                   // (no sequence, and the rows outside stay as they are)
    hipLaunchKernelGGL((rp_fwd_kernel<T, DT, QT>), dim3((unsigned)n), dim3(256), lds, s, a);
    const int rc2 = amdseg_launch_status();
    return rc2 ? rc2 : rp_join_launch<T>(a, s);
}
template <typename T>
static int rp_few_d(const RpArgs& a, hipStream_t s) {
    const int rc = a.D <= 32 ? rp_few_launch<T, 2>(a, s) : a.D <= 64 ? rp_few_launch<T, 4>(a, s) : a.D <= 96 ? rp_few_launch<T, 6>(a, s) : rp_few_launch<T, 8>(a, s);
    return rc ? rc : rp_join_launch<T>(a, s);
}
template <typename T, int QT>
static int rp_fwd_d(const RpArgs& a, hipStream_t s) {
    return a.D <= 32 ? rp_fwd_launch<T, 2, QT>(a, s) : a.D <= 64 ? rp_fwd_launch<T, 4, QT>(a, s) : a.D <= 96 ? rp_fwd_launch<T, 6, QT>(a, s)
                                                                                          : rp_fwd_launch<T, 8, QT>(a, s);
}
int amdseg_relpos_fwd_impl(const RpArgs& a0, int dtype, hipStream_t s) {
    RpArgs a = a0;
    if (rp_few(a)) return dtype == 1 ? rp_few_d<float>(a, s) : rp_few_d<bf16_t>(a, s);
    const int qt = rp_fwd_qt(a, dtype);
    rp_blocks(a, a.Lq, a.Tq, 64 * qt, a.heads);
    a.mask_words = rp_mask_bytes(a) / 8;
    if (dtype == 1) return rp_fwd_d<float, 1>(a, s);
    return qt == 1 ? rp_fwd_d<bf16_t, 1>(a, s) : rp_fwd_d<bf16_t, 2>(a, s);
}
