// The relative position bias as a dense tensor, for attention that is composed from single operations (dropout on the probabilities, returned
// probabilities), and its gradient:   bias[h, i, j] = table[map[clamp(j - i - off, -span, span) + span], h]
//                                     dtable[bk, h] = sum over b and (i, j) in bucket bk of dbias[b, h, i, j]
#include "relpos.h"
#include "relpos_launch.h"

// Write-bound.  A workgroup keeps its head's 2 span + 1 values in LDS (one float of gap per 8, so that lanes 8 elements apart hit different banks)
// and writes rows in 16-byte units; a row that does not start on 16 bytes has its first and last unit element by element.
// 12 x 1537 x 2049 fp32: 151 MB in 27 us, 5.7 TB/s; 12 x 512 x 512 bf16: 5.5 us.
template <typename T>
__global__ __launch_bounds__(256) void rp_bias_kernel(RpArgs a, int off, int rows_per_wg) {
    extern __shared__ float val[];
    constexpr int E = 16 / sizeof(T);
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, h = blockIdx.y;
    for (int x = tid; x <= 2 * a.span; x += 256) val[x + (x >> 3)] = rp_table(a, a.map[x], h);
    __syncthreads();
    const int i0 = blockIdx.x * rows_per_wg, i1 = min(i0 + rows_per_wg, a.Lq);
    for (int i = i0 + w; i < i1; i += 4) {
        const int64_t at = ((int64_t)h * a.Lq + i) * a.Lk;
        const int mis = (int)(at & (E - 1));                // (the tensor itself starts on 16 bytes)
        T* row = (T*)a.out + at;
        for (int u = l; u * E < mis + a.Lk; u += 64) {
            const int j = u * E - mis, x0 = j - i - off + a.span;
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) { const int x = rp_clamp(x0 + e, 0, 2 * a.span); v[e] = val[x + (x >> 3)]; }
            if (j >= 0 && j + E <= a.Lk) {
#pragma unroll
                for (int e = 0; e < E; e += 4) RpTile<T, 2>::st4(row + j + e, (f32x4){v[e], v[e + 1], v[e + 2], v[e + 3]});
            } else
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (j + e >= 0 && j + e < a.Lk) Act<T>::st(row + j + e, v[e]);
        }
    }
}

// Read-bound.  A workgroup takes a strip of rows of one (sequence, head).
//  * Places with |rel| < span, 8 x 8 blocks at a time: a lane owns a block diagonal and walks it down the strip (its wave takes every fourth block of it), so that
//    equal rel stay in the same one of its 15 registers; 16 bytes a load, 64 lanes side by side.  At the end the lanes lay their registers into LDS, the lower 8
//    first, then the upper 7, which belong to the next lane's places: one writer each, no order of arrival anywhere.
//  * The two far sides are one sum each: 16 lanes a row, 16-byte loads, four under way.
// 2 x 12 x 1537 x 2049 fp32 (rows that start on 4 bytes): 302 MB in 84 us, 3.6 TB/s, joins 9 us; 8 x 12 x 512 x 512 bf16 16 us, joins 9.
typedef uint32_t rp_u4 __attribute__((ext_vector_type(4), aligned(2)));      // 16 bytes from any element: rows start where they start
template <typename T> __device__ __forceinline__ void rp_ld8(const T* p, float (&v)[8]);
template <> __device__ __forceinline__ void rp_ld8<bf16_t>(const bf16_t* p, float (&v)[8]) {
    const rp_u4 q = *reinterpret_cast<const rp_u4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(q[i] << 16); v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u); }
}
template <> __device__ __forceinline__ void rp_ld8<float>(const float* p, float (&v)[8]) {
    const rp_u4 a = *reinterpret_cast<const rp_u4*>(p), b = *reinterpret_cast<const rp_u4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(a[i]); v[4 + i] = __uint_as_float(b[i]); }
}
__device__ __forceinline__ float rp_sum16(uint4 q, float) {
    return (__uint_as_float(q.x) + __uint_as_float(q.y)) + (__uint_as_float(q.z) + __uint_as_float(q.w));
}
__device__ __forceinline__ float rp_sum16(uint4 q, bf16_t) {
    const uint32_t v[4] = {q.x, q.y, q.z, q.w};
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += __uint_as_float(v[i] << 16) + __uint_as_float(v[i] & 0xffff0000u);
    return s;
}
template <typename T>
__global__ __launch_bounds__(256) void rp_bias_bwd_kernel(const T* d, float* part, int Lq, int Lk, int span, int off, int rows) {
    __shared__ float bins[4][64 * 8 + 8];
    __shared__ float red[2][4];
    constexpr int E = 16 / sizeof(T);
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, nd = 2 * span + 1, h = blockIdx.y, b = blockIdx.z, heads = gridDim.y;
    const int i0 = blockIdx.x * rows, i1 = min(i0 + rows, Lq);
    const int64_t plane = ((int64_t)b * heads + h) * Lq;
    float* out = part + (((int64_t)h * gridDim.z + b) * gridDim.x + blockIdx.x) * nd;
    // block diagonal n holds rel 8 n - span - 7 .. 8 n - span + 7, register e the e-th of them
    for (int n0 = 0; n0 * 8 <= 2 * span + 6; n0 += 64) {
        const int n = n0 + l, rel = 8 * n - span;           // rel of the block's main diagonal
        float acc[15];
#pragma unroll
        for (int e = 0; e < 15; ++e) acc[e] = 0.f;
        if (rel - 7 < span)
            for (int i = i0 + 8 * w; i < i1; i += 32) {
                const int j = i + off + rel;                // the block's first column
                if (j <= -8 || j >= Lk) continue;
                const T* p = d + (plane + i) * Lk + j;
                if (j >= 0 && j + 8 <= Lk && i + 8 <= i1) {
                    float v[8][8];
#pragma unroll
                    for (int r = 0; r < 8; ++r) rp_ld8<T>(p + (int64_t)r * Lk, v[r]);
#pragma unroll
                    for (int r = 0; r < 8; ++r)
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[7 + e - r] += v[r][e];
                } else
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (i + r < i1)
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (j + e >= 0 && j + e < Lk) acc[7 + e - r] += Act<T>::ld(p + (int64_t)r * Lk + e);
            }
        // place x of `out` is rel x - span; register e of block diagonal n is place 8 n - 7 + e
#pragma unroll
        for (int e = 0; e < 8; ++e) bins[w][8 * l + e] = acc[e];
        if (l == 63)
#pragma unroll
            for (int e = 0; e < 8; ++e) bins[w][512 + e] = 0.f;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 7; ++e) bins[w][8 * (l + 1) + e] += acc[8 + e];
        __syncthreads();
        for (int x = tid; x < 520; x += 256) {
            const int place = 8 * n0 - 7 + x;
            if (place >= 1 && place < nd - 1) {
                const float s = (bins[0][x] + bins[1][x]) + (bins[2][x] + bins[3][x]);
                // (the first 8 places of a later round of 64 diagonals have had the upper registers of the round before)
                out[place] = n0 > 0 && x < 8 ? out[place] + s : s;
            }
        }
        __syncthreads();
    }
    float sl = 0.f, sr = 0.f;
    const int l16 = tid & 15;
    for (int i = i0 + (tid >> 4); i < i1; i += 16) {
        const int64_t at = (plane + i) * Lk;
        const int mis = (int)(at & (E - 1));
        const T* row = d + at;
        const int jl = rp_clamp(i + off - span + 1, 0, Lk), jr = span == 0 ? jl : rp_clamp(i + off + span, 0, Lk);   // [0, jl) left, [jr, Lk) right
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const int ja = side ? jr : 0, jb = side ? Lk : jl;
            float s = 0.f;
            const int ua = (ja + mis + E - 1) / E, ub = (jb + mis) / E;           // whole 16-byte units
            const uint4* unit = reinterpret_cast<const uint4*>(row - mis);
            int u = ua + l16;
            for (; u + 48 < ub; u += 64) {
                const uint4 q0 = unit[u], q1 = unit[u + 16], q2 = unit[u + 32], q3 = unit[u + 48];
                s += (rp_sum16(q0, T(0)) + rp_sum16(q1, T(0))) + (rp_sum16(q2, T(0)) + rp_sum16(q3, T(0)));
            }
            for (; u < ub; u += 16) s += rp_sum16(unit[u], T(0));
            // the elements in front of the first whole unit and behind the last
            const int h1 = min(ua * E - mis, jb), t0 = max(ub * E - mis, h1);
            if (ja + l16 < h1) s += Act<T>::ld(row + ja + l16);
            if (t0 + l16 < jb) s += Act<T>::ld(row + t0 + l16);
            if (side) sr += s; else sl += s;
        }
    }
    sl = wave_sum(sl); sr = wave_sum(sr);
    if (l == 0) { red[0][w] = sl; red[1][w] = sr; }
    __syncthreads();
    if (tid == 0) {
        const float L = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]), R = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
        if (span == 0) out[0] = L + R;
        else { out[0] = L; out[nd - 1] = R; }
    }
}

static int rp_bias_rows(int64_t planes, int Lq) {           // rows of a strip: 64, less where that leaves CUs idle
    int rows = 64;
    while (rows > 16 && planes * ((Lq + rows - 1) / rows) < 1024) rows >>= 1;
    return rows;
}
size_t amdseg_relpos_bias_ws_impl(int B, int heads, int Lq, int span) {
    const int rows = rp_bias_rows((int64_t)B * heads, Lq);
    const size_t nd = 2 * (size_t)span + 1;
    return 4 * nd * heads * (1 + (size_t)B * ((Lq + rows - 1) / rows));
}
int amdseg_relpos_bias_fwd_impl(const RpArgs& a, int off, int dtype, hipStream_t s) {
    const int rows = rp_bias_rows(a.heads, a.Lq), lds = (2 * a.span + 1 + (2 * a.span + 1) / 8 + 1) * 4;
    const dim3 grid((a.Lq + rows - 1) / rows, a.heads);
    if (grid.x > RP_MAX_WGS) return AMDSEG_ERR_SHAPE;
    if (dtype == 1) hipLaunchKernelGGL((rp_bias_kernel<float>), grid, dim3(256), lds, s, a, off, rows);
    else hipLaunchKernelGGL((rp_bias_kernel<bf16_t>), grid, dim3(256), lds, s, a, off, rows);
    return amdseg_launch_status();
}
int amdseg_relpos_bias_bwd_impl(const void* d, int dtype, const int* map, int span, int buckets, int B, int heads, int Lq, int Lk, int off, float* dtable,
                                float* ws, hipStream_t s) {
    const int rows = rp_bias_rows((int64_t)B * heads, Lq), nd = 2 * span + 1;
    const dim3 grid((Lq + rows - 1) / rows, heads, B);
    if (grid.x > RP_MAX_WGS) return AMDSEG_ERR_SHAPE;
    float* part = ws + (size_t)nd * heads;
    if (B == 0) return amdseg_relpos_sums_impl(part, ws, 0, map, span, 0, buckets, heads, dtable, 0, s);       // nothing to sum: zeros
    if (dtype == 1) hipLaunchKernelGGL((rp_bias_bwd_kernel<float>), grid, dim3(256), 0, s, (const float*)d, part, Lq, Lk, span, off, rows);
    else hipLaunchKernelGGL((rp_bias_bwd_kernel<bf16_t>), grid, dim3(256), 0, s, (const bf16_t*)d, part, Lq, Lk, span, off, rows);
    int rc = amdseg_launch_status();
    if (rc) return rc;
    return amdseg_relpos_sums_impl(part, ws, (int64_t)B * grid.x, map, span, 0, buckets, heads, dtable, 0, s);
}
