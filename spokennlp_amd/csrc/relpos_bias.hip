// The relative position bias as a dense tensor, for attention that is composed from single operations (dropout on the probabilities, returned
// probabilities), and its gradient:   bias[h, i, j] = table[map[clamp(j - i - off, -span, span) + span], h]
//                                     dtable[bk, h] = sum over b and (i, j) in bucket bk of dbias[b, h, i, j]
#include "relpos.h"
#include "relpos_launch.h"

// Write-bound.  A workgroup keeps its head's 2 span + 1 values in LDS (one float of gap per 8, so that lanes 8 elements apart hit different banks)
// and writes rows in 16-byte units; a row that does not start on 16 bytes has its first and last unit element by element.
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

// Read-bound.  A workgroup takes a strip of rows of one (sequence, head).  Places with |rel| < span: a thread owns one rel and walks the rows -- neighbours
// read neighbouring elements, the sum stays in a register, no order of arrival anywhere.  The two far sides are one sum each: 16 lanes a row, 16-byte loads.
template <typename T>
__global__ __launch_bounds__(256) void rp_bias_bwd_kernel(const T* d, float* part, int Lq, int Lk, int span, int off, int rows) {
    __shared__ float red[2][4];
    constexpr int E = 16 / sizeof(T);
    const int tid = threadIdx.x, nd = 2 * span + 1, h = blockIdx.y, b = blockIdx.z, heads = gridDim.y;
    const int i0 = blockIdx.x * rows, i1 = min(i0 + rows, Lq);
    const int64_t plane = ((int64_t)b * heads + h) * Lq;
    float* out = part + (((int64_t)h * gridDim.z + b) * gridDim.x + blockIdx.x) * nd;
    for (int x = tid + 1; x < nd - 1; x += 256) {           // rel = x - span strictly inside
        const int rel = x - span;
        // rows with 0 <= i + off + rel < Lk
        const int a0 = max(i0, -off - rel), a1 = min(i1, Lk - off - rel);
        const T* p = d + (plane + a0) * Lk + (a0 + off + rel);
        float s = 0.f;
        int i = a0;
        for (; i + 8 <= a1; i += 8) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = Act<T>::ld(p + (int64_t)e * (Lk + 1));
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[e];
            p += (int64_t)8 * (Lk + 1);
        }
        for (; i < a1; ++i) { s += Act<T>::ld(p); p += Lk + 1; }
        out[x] = s;
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
            for (int u = (ja + mis) / E + l16; u * E - mis < jb; u += 16) {
                const int j = u * E - mis;
                if (j >= ja && j + E <= jb) {
                    const uint4 q = *reinterpret_cast<const uint4*>(row + j);
                    const uint32_t v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s += sizeof(T) == 2 ? __uint_as_float(v[e] << 16) + __uint_as_float(v[e] & 0xffff0000u) : __uint_as_float(v[e]);
                } else
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (j + e >= ja && j + e < jb) s += Act<T>::ld(row + j + e);
            }
            if (side) sr += s; else sl += s;
        }
    }
    sl = wave_sum(sl); sr = wave_sum(sr);
    if ((tid & 63) == 0) { red[0][tid >> 6] = sl; red[1][tid >> 6] = sr; }
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
    if (dtype == 1) hipLaunchKernelGGL((rp_bias_kernel<float>), grid, dim3(256), lds, s, a, off, rows);
    else hipLaunchKernelGGL((rp_bias_kernel<bf16_t>), grid, dim3(256), lds, s, a, off, rows);
    return amdseg_launch_status();
}
int amdseg_relpos_bias_bwd_impl(const void* d, int dtype, const int* map, int span, int buckets, int B, int heads, int Lq, int Lk, int off, float* dtable,
                                float* ws, hipStream_t s) {
    const int rows = rp_bias_rows((int64_t)B * heads, Lq), nd = 2 * span + 1;
    const dim3 grid((Lq + rows - 1) / rows, heads, B);
    float* part = ws + (size_t)nd * heads;
    if (B == 0) return amdseg_relpos_sums_impl(part, ws, 0, map, span, 0, buckets, heads, dtable, 0, s);       // nothing to sum: zeros
    if (dtype == 1) hipLaunchKernelGGL((rp_bias_bwd_kernel<float>), grid, dim3(256), 0, s, (const float*)d, part, Lq, Lk, span, off, rows);
    else hipLaunchKernelGGL((rp_bias_bwd_kernel<bf16_t>), grid, dim3(256), 0, s, (const bf16_t*)d, part, Lq, Lk, span, off, rows);
    int rc = amdseg_launch_status();
    if (rc) return rc;
    return amdseg_relpos_sums_impl(part, ws, (int64_t)B * grid.x, map, span, 0, buckets, heads, dtable, 0, s);
}
