// Distillation from a teacher's top logits (sm_100a): per row of student logits z
// (V entries) and K teacher logits t_j at columns i_j,
//   p = softmax(t / T) over the kept entries, q = softmax(z / T),
//   loss = T^2 sum_j p_j (log p_j - log q_{i_j}),  d loss / d z = T (q - p).
// Forward: one pass over z folds (max, sum-exp) of z / T; the K entries are
// gathered while it streams.  Backward: one read and one write of each element,
// then the K entries of the row are put right by the CTA that wrote them.
// Both are bound by memory: V elements per row read, and read and written.
#include "common.cuh"
#include "rows.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>

namespace fl {

template <>
struct Elem<__nv_bfloat16> {
    static constexpr int kPerVec = 8;
    __device__ __forceinline__ static float load1(const __nv_bfloat16* p) {
        return __uint_as_float(static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(p))) << 16);
    }
    __device__ __forceinline__ static void unpack(uint4 r, float* v) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

namespace {

constexpr int kMaxTop = 1024;
constexpr int kDThreads = 256;

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
__device__ __forceinline__ uint4 pack_vec(const float* v);
template <>
__device__ __forceinline__ uint4 pack_vec<float>(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                      __float_as_uint(v[3]));
}
template <>
__device__ __forceinline__ uint4 pack_vec<__half>(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ uint4 pack_vec<__nv_bfloat16>(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The teacher's entries: K per row, dense; dtype 0 fp32, 1 fp16, 2 bf16.
struct Teacher {
    const void* logits;
    const int64_t* index;
    int K, dtype;
    __device__ __forceinline__ float logit(int64_t row, int j) const {
        const int64_t i = row * K + j;
        if (dtype == 0) return __ldg(static_cast<const float*>(logits) + i);
        const uint16_t h = __ldg(static_cast<const uint16_t*>(logits) + i);
        if (dtype == 1) return __half2float(__ushort_as_half(h));
        return __uint_as_float(static_cast<uint32_t>(h) << 16);
    }
    __device__ __forceinline__ int64_t column(int64_t row, int j) const {
        return __ldg(index + row * K + j);
    }
};

// Padding entries (index -1) and entries of -inf carry no probability.
__device__ __forceinline__ bool kept(float t, int64_t column) { return column != -1 && t != -INFINITY; }

template <int K>
__device__ __forceinline__ void scale_by(float* v, float inv_t) {
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] *= inv_t;
}

// One warp forms the row's value from lse = LSE(z / T) and its own pass over the
// K entries; every lane ends with it, and with the teacher's lse (-inf: nothing kept).
template <typename T>
__device__ __forceinline__ float row_loss(const T* rowp, int64_t V, int64_t row, const Teacher& te,
                                          float lse, float inv_t, float t2, float& teacher_lse, bool& bad) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY, s = 0.0f;
    for (int j = lane; j < te.K; j += 32) {
        const float t = te.logit(row, j);
        if (kept(t, te.column(row, j))) ms_fold1(m, s, t * inv_t);
    }
    ms_warp_allreduce(m, s);
    teacher_lse = ms_finalize(m, s, -INFINITY);
    float sum = 0.0f;
    bool off = false;
    for (int j = lane; j < te.K; j += 32) {
        const float t = te.logit(row, j);
        const int64_t c = te.column(row, j);
        if (!kept(t, c)) continue;
        if (c < 0 || c >= V) {
            off = true;
            continue;
        }
        const float lp = t * inv_t - teacher_lse;
        const float p = ex2(lp * kLog2e);
        // log p - log q, taken as (t - z) / T - (teacher lse - lse): near a matched
        // student both differences are small and exact
        const float gap = (t * inv_t - Elem<T>::load1(rowp + c) * inv_t) - (teacher_lse - lse);
        if (p != 0.0f) sum += p * gap;  // 0 log 0 = 0, a NaN stays
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    bad = __any_sync(0xffffffffu, off);
    if (teacher_lse == -INFINITY) return 0.0f;
    return bad ? __int_as_float(0x7fc00000) : t2 * sum;
}

// A CTA per row segment, the nseg CTAs of a row in one cluster (as lse_segment_kernel).
template <typename T, bool SCALED>
__global__ void __launch_bounds__(kDThreads) distill_fwd_kernel(
    const T* __restrict__ x, int64_t V, RowMap rm, Teacher te, float inv_t, float t2, int nseg,
    float* __restrict__ lse_out, float* __restrict__ teacher_lse_out, float* __restrict__ values,
    int* __restrict__ err) {
    constexpr int E = Elem<T>::kPerVec, U = 4;
    __shared__ float2 seg[kMaxSeg];
    const int64_t row = blockIdx.x / nseg;
    const int rank = blockIdx.x % nseg;
    const T* rowp = x + rm(row);
    const int64_t head = head_elems(rowp, V), nv = (V - head) / E, tail0 = head + nv * E;
    const int64_t per = (nv + nseg - 1) / nseg;
    const int64_t v0 = min(nv, per * rank), v1 = min(nv, v0 + per);
    const uint4* vp = reinterpret_cast<const uint4*>(rowp + head);
    if (nseg > 1) cluster_arrive_relaxed();
    float m = -INFINITY, s = 0.0f;
    int64_t i = v0 + threadIdx.x;
    for (; i + (U - 1) * kDThreads < v1; i += U * kDThreads) {
        uint4 r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) r[u] = ld_stream_u4(vp + i + u * kDThreads);
        float v[U * E];
#pragma unroll
        for (int u = 0; u < U; ++u) Elem<T>::unpack(r[u], v + u * E);
        if (SCALED) scale_by<U * E>(v, inv_t);
        ms_fold<U * E>(m, s, v);
    }
    for (; i < v1; i += kDThreads) {
        float v[E];
        Elem<T>::unpack(ld_stream_u4(vp + i), v);
        if (SCALED) scale_by<E>(v, inv_t);
        ms_fold<E>(m, s, v);
    }
    if (rank == 0) {
        if (threadIdx.x < head) ms_fold1(m, s, Elem<T>::load1(rowp + threadIdx.x) * inv_t);
        if (tail0 + threadIdx.x < V) ms_fold1(m, s, Elem<T>::load1(rowp + tail0 + threadIdx.x) * inv_t);
    }
    ms_block_reduce<kDThreads>(m, s);
    if (nseg > 1) {
        cluster_wait();
        if (threadIdx.x == 0) {
            const uint32_t own = static_cast<uint32_t>(__cvta_generic_to_shared(&seg[rank]));
            uint32_t dst;
            asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(dst) : "r"(own));
            asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(m), "f"(s) : "memory");
        }
        asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (rank != 0) return;
    }
    if (threadIdx.x >= 32) return;
    if (nseg > 1) {
        m = seg[0].x, s = seg[0].y;
        for (int r = 1; r < nseg; ++r) ms_merge(m, s, seg[r].x, seg[r].y);
    } else {
        m = __shfl_sync(0xffffffffu, m, 0);
        s = __shfl_sync(0xffffffffu, s, 0);
    }
    const float lse = ms_finalize(m, s, -INFINITY);
    float tl;
    bool bad;
    const float value = row_loss(rowp, V, row, te, lse, inv_t, t2, tl, bad);
    if (threadIdx.x == 0) {
        lse_out[row] = lse;
        teacher_lse_out[row] = tl;
        values[row] = value;
        if (bad && err) atomicOr(err, 1);
    }
}

// Sum or mean (over the rows that keep an entry) in a fixed order, in 64 bits.
__global__ void __launch_bounds__(1024) distill_reduce_kernel(const float* __restrict__ values,
                                                              const float* __restrict__ teacher_lse,
                                                              int64_t N, int mean, float* __restrict__ out,
                                                              float* __restrict__ count_out) {
    __shared__ double sums[32];
    __shared__ int counts[32];
    double sum = 0.0;
    int count = 0;
    for (int64_t i = threadIdx.x; i < N; i += 1024) {
        sum += values[i];
        count += teacher_lse[i] != -INFINITY;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        count += __shfl_xor_sync(0xffffffffu, count, o);
    }
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum, counts[threadIdx.x >> 5] = count;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0, count = 0;
        for (int w = 0; w < 32; ++w) sum += sums[w], count += counts[w];
        *out = static_cast<float>(mean ? sum / count : sum);
        if (mean) *count_out = static_cast<float>(count);
    }
}

// dz = c (q - p), c = g T: a CTA takes one chunk of one row, writes c q, then
// rewrites the chunk's teacher columns with every entry of theirs taken off in fp32.
template <typename T>
__global__ void __launch_bounds__(kDThreads) distill_bwd_kernel(
    const float* __restrict__ g, int scalar_g, const float* __restrict__ count, float temp,
    const T* __restrict__ x, int64_t V, RowMap rm, Teacher te, float inv_t,
    const float* __restrict__ lse_in, const float* __restrict__ teacher_lse_in, T* __restrict__ gx,
    int nchunk, int64_t chunk_vec) {
    constexpr int E = Elem<T>::kPerVec, U = 4;
    __shared__ int fix_col[kMaxTop];
    __shared__ float fix_p[kMaxTop];
    __shared__ int fix_n;
    const int chunk = blockIdx.x % nchunk;
    const int64_t row = blockIdx.x / nchunk;
    const T* rowp = x + rm(row);
    T* outp = gx + row * V;
    const float lse = __ldg(lse_in + row), tl = __ldg(teacher_lse_in + row);
    const bool live = tl != -INFINITY;
    float c = scalar_g ? __ldg(g) : __ldg(g + row);
    if (count) c /= __ldg(count);
    c *= temp;
    const int64_t head = head_elems(rowp, V), nv = (V - head) / E, tail0 = head + nv * E;
    const int64_t v0 = min(nv, chunk * chunk_vec), v1 = min(nv, v0 + chunk_vec);
    auto q = [&](float z) { return live ? c * exp_from(z * inv_t, lse) : 0.0f; };
    // this chunk's columns (the first chunk has the head, the last the tail)
    const int64_t c0 = chunk == 0 ? 0 : head + v0 * E;
    const int64_t c1 = chunk == nchunk - 1 ? V : head + v1 * E;
    if (threadIdx.x == 0) fix_n = 0;
    __syncthreads();
    if (live) {
        for (int j = threadIdx.x; j < te.K; j += kDThreads) {
            const int64_t col = te.column(row, j);
            if (col >= c0 && col < c1) {
                const float t = te.logit(row, j);
                if (t != -INFINITY) {
                    const int at = atomicAdd(&fix_n, 1);
                    fix_col[at] = static_cast<int>(col - c0);
                    fix_p[at] = ex2((t * inv_t - tl) * kLog2e);
                }
            }
        }
    }
    if (chunk == 0 && threadIdx.x < head)
        outp[threadIdx.x] = narrow<T>(q(Elem<T>::load1(rowp + threadIdx.x)));
    if (chunk == nchunk - 1 && tail0 + threadIdx.x < V)
        outp[tail0 + threadIdx.x] = narrow<T>(q(Elem<T>::load1(rowp + tail0 + threadIdx.x)));
    const uint4* vp = reinterpret_cast<const uint4*>(rowp + head);
    if (((reinterpret_cast<uintptr_t>(rowp) ^ reinterpret_cast<uintptr_t>(outp)) & 15u) == 0) {
        uint4* op = reinterpret_cast<uint4*>(outp + head);
        auto vec = [&](uint4 r) {
            float v[E];
            Elem<T>::unpack(r, v);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = q(v[e]);
            return pack_vec<T>(v);
        };
        int64_t i = v0 + threadIdx.x;
        for (; i + (U - 1) * kDThreads < v1; i += U * kDThreads) {
            uint4 r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) r[u] = ld_stream_u4(vp + i + u * kDThreads);
#pragma unroll
            for (int u = 0; u < U; ++u) __stcs(op + i + u * kDThreads, vec(r[u]));
        }
        for (; i < v1; i += kDThreads) __stcs(op + i, vec(ld_stream_u4(vp + i)));
    } else {
        // x and gx rows start at different phases of 16 bytes: element by element
        for (int64_t e = head + v0 * E + threadIdx.x; e < head + v1 * E; e += kDThreads)
            outp[e] = narrow<T>(q(Elem<T>::load1(rowp + e)));
    }
    __syncthreads();
    const int n = fix_n;
    for (int j = threadIdx.x; j < n; j += kDThreads) {
        // entries of one column: the largest probability leads (ties: any, they are
        // equal), and sums them from the largest down, an order their list has no part in
        const int col = fix_col[j];
        bool lead = true;
        float sum = fix_p[j];
        int same = 0;
        for (int k = 0; k < n; ++k)
            if (fix_col[k] == col && k != j) {
                ++same;
                if (fix_p[k] > fix_p[j] || (fix_p[k] == fix_p[j] && k < j)) lead = false;
            }
        if (!lead) continue;
        if (same) {
            float last = fix_p[j];
            int used_at = j;
            for (int r = 0; r < same; ++r) {
                float best = -1.0f;
                int at = -1;
                for (int k = 0; k < n; ++k) {
                    if (fix_col[k] != col || k == j) continue;
                    const bool after = fix_p[k] < last || (fix_p[k] == last && k > used_at);
                    if (after && (fix_p[k] > best || (fix_p[k] == best && k < at))) best = fix_p[k], at = k;
                }
                if (at < 0) break;  // NaN probabilities: the sum is NaN already
                sum += best;
                last = best;
                used_at = at;
            }
        }
        const int64_t e = c0 + col;
        outp[e] = narrow<T>(c * (exp_from(Elem<T>::load1(rowp + e) * inv_t, lse) - sum));
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check_distill(const void* x, int dtype, const void* tlogits, int tdtype, const int64_t* index, int64_t N,
                  int64_t V, int64_t K, float temperature, const char* what) {
    FL_REQUIRE(N >= 0 && V >= 1 && K >= 1, "%s: bad shape (%lld, %lld), %lld teacher entries", what,
               (long long)N, (long long)V, (long long)K);
    FL_REQUIRE(K <= kMaxTop, "%s: at most %d teacher entries", what, kMaxTop);
    FL_REQUIRE(V <= INT32_MAX, "%s: V too large", what);
    FL_REQUIRE(dtype >= 0 && dtype <= 2 && tdtype >= 0 && tdtype <= 2, "%s: unknown dtype", what);
    FL_REQUIRE(temperature > 0.0f && temperature <= 3.0e38f, "%s: temperature must be positive", what);
    FL_REQUIRE(N == 0 || (x && tlogits && index), "%s: NULL buffer", what);
    FL_REQUIRE(aligned_to(x, dtype == 0 ? 4 : 2) && aligned_to(tlogits, tdtype == 0 ? 4 : 2) &&
                   aligned_to(index, 8),
               "%s: misaligned buffer", what);
    return FL_OK;
}

int distill_rows(int64_t N, int64_t V, int64_t rows_per_group, int64_t group_stride, int64_t row_stride,
                 RowMap* rm, const char* what) {
    *rm = RowMap::dense(V);
    if (rows_per_group < 0) return FL_OK;
    FL_REQUIRE(rows_per_group >= 1 && group_stride >= 0 && row_stride >= 0, "%s: bad row layout", what);
    *rm = RowMap{rows_per_group, group_stride, row_stride};
    return FL_OK;
}

template <typename T>
int launch_fwd(const void* x, int64_t N, int64_t V, RowMap rm, Teacher te, float temp, float* lse,
               float* tlse, float* values, int* err, cudaStream_t s, const char* what) {
    // rows that cannot fill the SMs are split over a cluster, at least 32 KB to a CTA
    const int64_t target = 2ll * sm_count(), bytes = V * (int64_t)sizeof(T);
    int64_t nseg = N >= target ? 1 : (target + N - 1) / N;
    nseg = std::max<int64_t>(1, std::min<int64_t>({nseg, bytes / 32768, (int64_t)kMaxSeg}));
    FL_REQUIRE(N * nseg <= INT32_MAX, "%s: too many rows", what);
    LaunchCfg lc(dim3((unsigned)(N * nseg)), dim3(kDThreads), 0, s, false);
    lc.cluster((int)nseg);
    auto kern = temp == 1.0f ? distill_fwd_kernel<T, false> : distill_fwd_kernel<T, true>;
    FL_CUDA(cudaLaunchKernelEx(&lc.cfg, kern, static_cast<const T*>(x), V, rm, te, 1.0f / temp, temp * temp,
                               (int)nseg, lse, tlse, values, err));
    return check_launch(what);
}

template <typename T>
int launch_bwd(const float* g, int scalar_g, const float* count, const void* x, int64_t N, int64_t V,
               RowMap rm, Teacher te, float temp, const float* lse, const float* tlse, void* gx,
               cudaStream_t s, const char* what) {
    const int64_t nv = V * (int64_t)sizeof(T) / 16 + 1, chunk = 1024;
    const int64_t nchunk = (nv + chunk - 1) / chunk;
    FL_REQUIRE(N <= INT32_MAX / nchunk, "%s: too many rows", what);
    LaunchCfg lc(dim3((unsigned)(N * nchunk)), dim3(kDThreads), 0, s, false);
    FL_CUDA(cudaLaunchKernelEx(&lc.cfg, distill_bwd_kernel<T>, g, scalar_g, count, temp,
                               static_cast<const T*>(x), V, rm, te, 1.0f / temp, lse, tlse,
                               static_cast<T*>(gx), (int)nchunk, chunk));
    return check_launch(what);
}

}  // namespace
}  // namespace fl

using namespace fl;

extern "C" int fl_topk_distill_fwd(const void* x, int dtype, const void* teacher_logits, int teacher_dtype,
                                   const int64_t* teacher_index, int64_t N, int64_t V, int64_t K,
                                   int64_t rows_per_group, int64_t group_stride, int64_t row_stride,
                                   float temperature, int reduce, float* lse, float* teacher_lse,
                                   float* values, float* out, float* count, int* err_flag,
                                   fl_stream_t stream) {
    clear_error();
    const char* what = "fl_topk_distill_fwd";
    if (int st = check_distill(x, dtype, teacher_logits, teacher_dtype, teacher_index, N, V, K, temperature, what))
        return st;
    RowMap rm;
    if (int st = distill_rows(N, V, rows_per_group, group_stride, row_stride, &rm, what)) return st;
    FL_REQUIRE(reduce >= 1 && reduce <= 3, "%s: unknown reduction %d", what, reduce);
    if (N == 0) return FL_OK;
    FL_REQUIRE(lse && teacher_lse && values && (reduce == 1 || out) && (reduce != 3 || count), "%s: NULL buffer", what);
    FL_REQUIRE(aligned_to(lse, 4) && aligned_to(teacher_lse, 4) && aligned_to(values, 4) &&
                   aligned_to(out, 4) && aligned_to(count, 4) && aligned_to(err_flag, 4),
               "%s: misaligned buffer", what);
    if (int st = bind_device(stream, lse)) return st;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const Teacher te{teacher_logits, teacher_index, (int)K, teacher_dtype};
    int st;
    if (dtype == 0)
        st = launch_fwd<float>(x, N, V, rm, te, temperature, lse, teacher_lse, values, err_flag, s, what);
    else if (dtype == 1)
        st = launch_fwd<__half>(x, N, V, rm, te, temperature, lse, teacher_lse, values, err_flag, s, what);
    else
        st = launch_fwd<__nv_bfloat16>(x, N, V, rm, te, temperature, lse, teacher_lse, values, err_flag, s, what);
    if (st || reduce == 1) return st;
    LaunchCfg lc(dim3(1), dim3(1024), 0, s, false);
    FL_CUDA(cudaLaunchKernelEx(&lc.cfg, distill_reduce_kernel, (const float*)values, (const float*)teacher_lse,
                               N, reduce == 3, out, count));
    return check_launch(what);
}

extern "C" int fl_topk_distill_bwd(const float* grad, const void* x, int dtype, const void* teacher_logits,
                                   int teacher_dtype, const int64_t* teacher_index, int64_t N, int64_t V,
                                   int64_t K, int64_t rows_per_group, int64_t group_stride,
                                   int64_t row_stride, float temperature, int reduce, const float* lse,
                                   const float* teacher_lse, const float* count, void* gx,
                                   fl_stream_t stream) {
    clear_error();
    const char* what = "fl_topk_distill_bwd";
    if (int st = check_distill(x, dtype, teacher_logits, teacher_dtype, teacher_index, N, V, K, temperature, what))
        return st;
    RowMap rm;
    if (int st = distill_rows(N, V, rows_per_group, group_stride, row_stride, &rm, what)) return st;
    FL_REQUIRE(reduce >= 1 && reduce <= 3, "%s: unknown reduction %d", what, reduce);
    if (N == 0) return FL_OK;
    FL_REQUIRE(grad && lse && teacher_lse && gx && (reduce != 3 || count), "%s: NULL buffer", what);
    FL_REQUIRE(aligned_to(grad, 4) && aligned_to(lse, 4) && aligned_to(teacher_lse, 4) &&
                   aligned_to(count, 4) && aligned_to(gx, dtype == 0 ? 4 : 2),
               "%s: misaligned buffer", what);
    if (int st = bind_device(stream, gx)) return st;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const Teacher te{teacher_logits, teacher_index, (int)K, teacher_dtype};
    const float* cnt = reduce == 3 ? count : nullptr;
    const int scalar = reduce != 1;
    if (dtype == 0)
        return launch_bwd<float>(grad, scalar, cnt, x, N, V, rm, te, temperature, lse, teacher_lse, gx, s, what);
    if (dtype == 1)
        return launch_bwd<__half>(grad, scalar, cnt, x, N, V, rm, te, temperature, lse, teacher_lse, gx, s, what);
    return launch_bwd<__nv_bfloat16>(grad, scalar, cnt, x, N, V, rm, te, temperature, lse, teacher_lse, gx, s, what);
}
