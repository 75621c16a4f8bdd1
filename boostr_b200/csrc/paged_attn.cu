// Attention over a paged key-value cache, one warp for each query head of each row: the plain form of the running softmax.
#include "paged.cuh"

namespace b200q {
namespace {

__global__ void __launch_bounds__(128) attn_row_kernel(const AttnParams p) {
    grid_dep_wait();
    grid_dep_launch();
    const uint64_t w = (uint64_t)blockIdx.x * 4 + threadIdx.x / 32;
    const uint32_t lane = threadIdx.x & 31;
    if (w >= (uint64_t)p.rows * p.hq) return;
    const uint32_t r = (uint32_t)(w / p.hq), h = (uint32_t)(w % p.hq);
    const uint32_t b = p.cu ? request_of(p.cu, p.requests, r) : r;
    const uint32_t len = attn_len(p, b);
    // position of the row: the rows of a request are the last of its tokens; rows behind the last request see nothing
    const int64_t pos = !p.cu ? (int64_t)len - 1 : (int64_t)r < p.cu[p.requests] ? (int64_t)len - p.cu[b + 1] + r : -1;
    const int64_t first = p.window && pos + 1 > p.window ? pos + 1 - p.window : 0;
    float q[8], o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t e = 64 * (i / 2) + 2 * lane + i % 2;
        q[i] = e < p.dim ? load_f32(p.q, (int64_t)r * p.q_row + (int64_t)h * p.q_head + e, p.q_dtype) * p.scale_log2 : 0.f;
        o[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int dt = p.f16 ? DT_F16 : DT_BF16;
    for (int64_t j = 0; j <= pos; ++j) {
        if (j < first && j >= p.sinks) j = first;
        uint32_t page, tok;
        if (!attn_page(p, b, (uint32_t)j, page, tok)) continue;
        const int64_t ka = (int64_t)page * p.k_page + (int64_t)tok * p.k_tok + (int64_t)(h / p.group) * p.k_head;
        const int64_t va = (int64_t)page * p.v_page + (int64_t)tok * p.v_tok + (int64_t)(h / p.group) * p.v_head;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t e = 64 * (i / 2) + 2 * lane + i % 2;
            if (e < p.dim) s = fmaf(q[i], load_f32(p.k, ka + e, dt), s);
        }
#pragma unroll
        for (int d = 1; d < 32; d *= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
        const float m2 = fmaxf(m, s), c = m2 == -INFINITY ? 1.f : exp2f(m - m2), e2 = m2 == -INFINITY ? 0.f : exp2f(s - m2);
        m = m2;
        l = fmaf(l, c, e2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t e = 64 * (i / 2) + 2 * lane + i % 2;
            if (e < p.dim) o[i] = fmaf(o[i], c, e2 * load_f32(p.v, va + e, dt));
        }
    }
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // a row that sees no key is zero
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t e = 64 * (i / 2) + 2 * lane + i % 2;
        if (e < p.dim) store_f32(p.out, ((int64_t)r * p.hq + h) * p.dim + e, p.out_dtype, o[i] * inv);
    }
    if (p.lse && lane == 0) p.lse[(int64_t)r * p.hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace

cudaError_t launch_attn_rows(const AttnParams& p, cudaStream_t st) {
    const uint64_t warps = (uint64_t)p.rows * p.hq;
    note_launch();
    return launch_pdl(attn_row_kernel, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, st, p);
}

}  // namespace b200q
