// Attention over the paged 4-bit cache (l3m_kv4_attend_dev; contract in include/l3m_kernels.h, layout in
// kv4.cuh).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <cmath>
#include <cstdio>
#include "kv4.cuh"

using namespace l3m;

extern "C" int l3m_error_msg(const char *msg);
extern "C" int l3m_error_cuda(int e, const char *what);

namespace {

int refuse(const char *entry, const char *why) {
    char msg[200];
    snprintf(msg, sizeof msg, "%s: %s", entry, why);
    return l3m_error_msg(msg);
}

struct AttendArgs {
    l3m_kv4_attend a;
    Kv4Dev c;
    int mx;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float *p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

__device__ __forceinline__ float code_value(unsigned nib, int mx) {
    if (!mx) return (float)(int)nib - 8.0f;
    const float m = (float)((0xC8643210u >> (4 * (nib & 7))) & 15) * 0.5f;
    return nib & 8 ? -m : m;
}
__device__ __forceinline__ float scale_value(const uint8_t *p, int mx) {
    return mx ? (*p ? __uint_as_float((uint32_t)*p << 23) : __uint_as_float(0x00400000u)) : __half2float(*(const __half *)p);
}

// One warp per query row, one cached token at a time: lane l holds dims l + 32 j. The softmax runs with the
// row's running maximum and sum.
template <typename T>
__global__ void __launch_bounds__(256) attend_rows(const AttendArgs p) {
    const l3m_kv4_attend &a = p.a;
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)a.max_q * a.n_req * a.n_heads;
    for (long long i = blockIdx.x * 8LL + (threadIdx.x >> 5); i < rows; i += gridDim.x * 8LL) {
        const int h = (int)(i % a.n_heads);
        const int r = (int)(i / a.n_heads % a.n_req), q = (int)(i / a.n_heads / a.n_req);
        const int start = a.q_start[r], nq = a.q_start[r + 1] - start;
        if (q >= nq) continue;
        const int kv = min(max(a.kv_len[r], 0), a.max_kv), pos = kv - nq + q;
        const int lo = a.window ? max(0, pos - a.window + 1) : 0;
        const int kh = h / (a.n_heads / p.c.n_kv), ng = p.c.ng, jt = (lane >> 3) * ng, gt = (lane >> 2) * ng;
        const T *qp = (const T *)a.q + (size_t)(start + q) * a.q_ld + (size_t)h * p.c.dim;
        float x[8], o[8] = {}, m = -INFINITY, l = 0.0f;
        for (int j = 0; j < ng; j++) x[j] = lane + 32 * j < p.c.dim ? to_f32(qp[lane + 32 * j]) * a.scale : 0.0f;
        for (int t = lo; t <= pos; t++) {
            const int id = a.tables[(size_t)r * a.max_blocks + t / p.c.page], off = t % p.c.page, tr = off % kKvTile;
            if (id < 0 || id >= p.c.n_pages) {
                if (a.status && lane == 0) atomicOr((int *)a.status, L3M_KV4_BAD_PAGE);
                continue;
            }
            const uint8_t *tile = p.c.data + p.c.tile_at(id, kh, off / kKvTile);
            float s = 0.0f;
            for (int j = 0; j < ng; j++) {
                const uint8_t b = tile[tr * 16 * ng + (jt + j) * 4 + (lane & 7) / 2];
                s = fmaf(x[j], code_value(lane & 1 ? b >> 4 : b & 15, p.mx) * scale_value(tile + p.c.k_scales() + (tr * ng + j) * p.c.sb, p.mx), s);
            }
            for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            const float mn = fmaxf(m, s), fix = m == -INFINITY ? 0.0f : expf(m - mn), w = expf(s - mn);
            m = mn;
            l = fmaf(l, fix, w);
            for (int j = 0; j < ng; j++) {
                const uint8_t b = tile[256 * ng + tr * 16 * ng + (gt + j) * 2 + (lane & 3) / 2];
                const float v = code_value(lane & 1 ? b >> 4 : b & 15, p.mx) * scale_value(tile + p.c.v_scales() + (tr * ng + j) * p.c.sb, p.mx);
                o[j] = fmaf(w, v, o[j] * fix);
            }
        }
        T *op = (T *)a.out + (size_t)(start + q) * a.out_ld + (size_t)h * p.c.dim;
        for (int j = 0; j < ng; j++)
            if (lane + 32 * j < p.c.dim) from_f32(op + lane + 32 * j, l > 0.0f ? o[j] / l : 0.0f);
    }
}

const char *attend_error(const l3m_kv4 *c, const l3m_kv4_attend *a) {
    if (const char *why = kv4_shape_error(c)) return why;
    if (!a) return "arguments are required";
    if (a->dtype != L3M_DT_F32 && a->dtype != L3M_DT_BF16) return "dtype must be f32 or bf16";
    if (a->n_heads < 1 || a->n_heads > 65535 || a->n_heads % c->n_kv_heads) return "n_heads must be a positive multiple of n_kv_heads";
    if (a->n_req < 0 || a->max_blocks < 0 || a->max_q < 0 || a->max_kv < 0 || a->window < 0) return "a count is negative";
    if (a->max_kv > (int64_t)a->max_blocks * c->page) return "max_kv must not exceed max_blocks * page";
    return nullptr;
}

}  // namespace

extern "C" {

L3M_API size_t l3m_kv4_attend_scratch(const l3m_kv4 *cache, const l3m_kv4_attend *a) {
    if (attend_error(cache, a)) return 0;
    return 16;
}

L3M_API int l3m_kv4_attend_dev(const l3m_kv4 *cache, const l3m_kv4_attend *a, void *stream) {
    const char *me = "l3m_kv4_attend_dev";
    if (const char *why = attend_error(cache, a)) return refuse(me, why);
    if (const char *why = kv4_error(cache)) return refuse(me, why);
    if (!std::isfinite(a->scale)) return refuse(me, "scale must be finite");
    if (!a->n_req || !a->max_q) return 0;
    if (!a->q || !a->out || !a->q_start || !a->kv_len || (a->max_blocks && !a->tables)) return refuse(me, "a pointer is missing");
    const int64_t width = (int64_t)a->n_heads * cache->head_dim;
    if (a->q_ld < width || a->out_ld < width) return refuse(me, "a token stride is smaller than its heads");
    if (((uintptr_t)a->q | (uintptr_t)a->out) & (a->dtype == L3M_DT_F32 ? 3 : 1) || ((uintptr_t)a->q_start | (uintptr_t)a->kv_len | (uintptr_t)a->tables) & 3)
        return refuse(me, "a pointer is not aligned to its type");
    if (!a->scratch || a->scratch_bytes < l3m_kv4_attend_scratch(cache, a) || ((uintptr_t)a->scratch & 15)) return refuse(me, "scratch is too small or not 16-byte aligned");
    const AttendArgs p = {*a, kv4_dev(cache), cache->dtype == L3M_DT_MXFP4};
    const long long rows = (long long)a->max_q * a->n_req * a->n_heads;
    const int grid = (int)std::min<long long>(148 * 16, (rows + 7) / 8);
    if (a->dtype == L3M_DT_F32) attend_rows<float><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
    else attend_rows<__nv_bfloat16><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : l3m_error_cuda(e, me);
}

}  // extern "C"
