// Attention of one new token per request over a paged cache: out = softmax(scale q K^T) V, by one pass over the visible keys
// and values with the running maximum and sum of the softmax.
//
// Bound: HBM reads of the keys and values (two bytes an element for 2 group flops each; the group's query heads share every
// byte).  The keys that a request sees (its sinks, then its window) are numbered through without a gap, cut into tiles of
// 64, and all tiles of the batch, request by request and head by head, are laid end to end; every CTA takes an equal run of
// them, so ragged batches and single long requests are balanced alike and the lengths are needed on the GPU only.
// Where a run ends inside a head, the CTAs that share the head leave partial sums in scratch, and the one that finishes last
// adds them up in their order (the result does not depend on which one that is).
//
// In a tile each of four warps owns 16 keys, with a ring of its own filled by asynchronous 16-byte copies (zeros where a key
// is not visible, so nothing that lies in unused places of a page can reach a sum); no barrier separates the warps until
// their sums are joined at the end of a head.  Products on mma.sync with the keys as the 16 rows and 8 query heads as the
// columns: S^T = K Q^T, O^T = V^T P^T; at two flops a byte and head the tensor cores idle at any rate, and the operands come
// straight from the 16-byte chunks that were copied.
#include "paged.cuh"

namespace b200q {

struct DecodePlan {
    uint32_t chunks;      // of up to 8 NT query heads that share a key-value head
    uint32_t items;       // hkv * chunks: what a request's keys are read for
    uint32_t min_tiles;   // of a CTA's run, where there are that many
    float* part;          // [2 grid] partial sums: O [8 NT][DP], then m [8 NT], l [8 NT]
    uint32_t* counters;   // [grid] zero between calls
};

namespace {

constexpr size_t DEC_COUNTER_BYTES = 4096;  // one counter for each CTA, zero between calls
constexpr int DEC_WARPS = 4, DEC_THREADS = 32 * DEC_WARPS, DEC_TILE = 16 * DEC_WARPS;

// f16 weights are kept 2^14 times their size: their subnormals would otherwise lose the small ones of a long row
template <bool F16>
constexpr float WEIGHT_BIAS = F16 ? 14.f : 0.f;

struct TileMeta {
    int valid;            // keys of the warp's 16 that are visible
    uint32_t b, h, h0;    // request, key-value head, first of the query heads that share it
    uint32_t t, nt;       // tile of its item, and their number
};

template <int DP, int NT, bool F16, bool SPLIT>
struct DecodeShape {
    static constexpr int KS = DP / 16, TERMS = SPLIT ? (F16 ? 2 : 3) : 1, HEADS = 8 * NT;
    static constexpr int ROW = DP * 2, WARP_STAGE = 2 * 16 * ROW, STAGE = DEC_WARPS * WARP_STAGE;
    static constexpr int STAGES = DP == 64 ? 4 : 3;
    static constexpr int Q_BYTES = KS * TERMS * NT * 32 * 8;
    static constexpr int OFF_Q = STAGES * STAGE, OFF_ML = OFF_Q + Q_BYTES, OFF_META = OFF_ML + DEC_WARPS * HEADS * 8,
                         SMEM = OFF_META + DEC_WARPS * STAGES * (int)sizeof(TileMeta);
    static constexpr int PART = HEADS * (DP + 2);  // floats of a partial sum
};

// Keys that request b's new token sees: [0, sinks) and [from, len), numbered through.
__device__ __forceinline__ void visible_keys(const AttnParams& p, uint32_t len, uint32_t& sinks, uint32_t& from, uint32_t& n) {
    from = p.window && len > p.window ? len - p.window : 0;
    sinks = min(p.sinks, from);
    n = sinks + (len - from);
}

// Elements dim .. dim + 3 of a row from its sums, and its log-sum-exp.  A sum of zero (every visible score is minus infinity)
// gives zeros.
template <bool F16>
__device__ __forceinline__ void write_row(const AttnParams& p, uint32_t b, uint32_t head, uint32_t dim, float4 a, float mx, float sum) {
    const int64_t row = (int64_t)b * p.hq + head;
    if (dim == 0 && p.lse) p.lse[row] = sum == 0.f ? -INFINITY : (mx - WEIGHT_BIAS<F16> + log2f(sum)) * 0.6931471805599453f;
    if (dim >= p.dim) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const float x[4] = {a.x * inv, a.y * inv, a.z * inv, a.w * inv};
    const int64_t at = row * p.dim + dim;
    if (p.out_dtype == DT_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        const uint2 r = p.out_dtype == DT_F16 ? make_uint2(pack2<true>(x[0], x[1]), pack2<true>(x[2], x[3]))
                                              : make_uint2(pack2<false>(x[0], x[1]), pack2<false>(x[2], x[3]));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = r;
    }
}

template <int DP, int NT, bool F16, bool SPLIT, int MINB>
__global__ void __launch_bounds__(DEC_THREADS, MINB) decode_kernel(const AttnParams p, const DecodePlan d) {
    using Sh = DecodeShape<DP, NT, F16, SPLIT>;
    constexpr int KS = Sh::KS, TERMS = Sh::TERMS, STAGES = Sh::STAGES, ROW = Sh::ROW, HEADS = Sh::HEADS;
    constexpr int CPR = ROW / 16, ROWS_PER = 32 / CPR > 0 ? 32 / CPR : 1;  // 16-byte chunks of a row; rows of one copy instruction
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sbase = smem_u32(smem);
    uint2* qf = reinterpret_cast<uint2*>(smem + Sh::OFF_Q);
    float2* ml = reinterpret_cast<float2*>(smem + Sh::OFF_ML);
    TileMeta* meta = reinterpret_cast<TileMeta*>(smem + Sh::OFF_META) + warp * STAGES;
    __shared__ uint64_t s_scan[DEC_WARPS];
    __shared__ uint32_t s_first[2];
    __shared__ uint32_t s_last;

    grid_dep_wait();
    grid_dep_launch();

    // ---- this CTA's run of tiles
    uint64_t begin, end, total;
    uint32_t active;
    {
        const uint32_t chunk = (p.requests + DEC_THREADS - 1) / DEC_THREADS;
        const uint32_t b0 = min(p.requests, threadIdx.x * chunk), b1 = min(p.requests, b0 + chunk);
        uint64_t sum = 0;
        for (uint32_t b = b0; b < b1; ++b) {
            uint32_t sk, fr, n;
            visible_keys(p, attn_len(p, b), sk, fr, n);
            sum += (n + DEC_TILE - 1) / DEC_TILE;
        }
        uint64_t s = sum;
#pragma unroll
        for (int i = 1; i < 32; i *= 2) {
            const uint64_t o = __shfl_up_sync(0xFFFFFFFFu, s, i);
            if (lane >= i) s += o;
        }
        if (lane == 31) s_scan[warp] = s;
        __syncthreads();
        uint64_t before = 0;
        total = 0;
#pragma unroll
        for (int w = 0; w < DEC_WARPS; ++w) {
            if (w < warp) before += s_scan[w];
            total += s_scan[w];
        }
        total *= d.items;
        const uint64_t runs = (total + d.min_tiles - 1) / d.min_tiles;
        active = (uint32_t)min((uint64_t)gridDim.x, runs);
        begin = end = 0;
        if (blockIdx.x < active) {
            begin = blockIdx.x * total / active;
            end = (blockIdx.x + 1ull) * total / active;
        }
        uint64_t pre = (before + s - sum) * d.items;  // tiles before request b0
        if (begin < end && begin >= pre && begin < pre + sum * d.items) {
            for (uint32_t b = b0; b < b1; ++b) {
                uint32_t sk, fr, n;
                visible_keys(p, attn_len(p, b), sk, fr, n);
                const uint64_t t = (uint64_t)((n + DEC_TILE - 1) / DEC_TILE) * d.items;
                if (begin < pre + t) {
                    s_first[0] = b;
                    s_first[1] = (uint32_t)(begin - pre);
                    break;
                }
                pre += t;
            }
        }
        __syncthreads();
    }
    // requests that see nothing
    for (uint32_t b = blockIdx.x; b < p.requests; b += gridDim.x)
        if (p.lens[b] <= 0) {
            for (uint32_t i = threadIdx.x; i < p.hq * p.dim; i += DEC_THREADS) store_f32(p.out, (int64_t)b * p.hq * p.dim + i, p.out_dtype, 0.f);
            if (p.lse)
                for (uint32_t i = threadIdx.x; i < p.hq; i += DEC_THREADS) p.lse[(int64_t)b * p.hq + i] = -INFINITY;
        }
    if (begin >= end) return;
    const uint32_t ntiles = (uint32_t)(end - begin);

    // ---- the cursor of the copies: the next tile whose page numbers are fetched
    uint32_t c_b = s_first[0], c_h, c_h0, c_t, c_nt, c_sinks, c_from, c_n, c_left = ntiles;
    visible_keys(p, attn_len(p, c_b), c_sinks, c_from, c_n);
    c_nt = (c_n + DEC_TILE - 1) / DEC_TILE;
    c_t = s_first[1] % c_nt;
    c_h = s_first[1] / c_nt / d.chunks;
    c_h0 = (s_first[1] / c_nt - c_h * d.chunks) * HEADS;
    // page and place in it of key lane % 16 of the warp's 16 in the next tile (page < 0: not visible).  Read one tile ahead and
    // not looked at before its copies are issued, so that no step waits for the table.
    int32_t page = -1;
    uint32_t tok = 0;
    TileMeta next;
    auto fetch = [&]() {
        page = -1;
        if (c_left == 0) return;
        --c_left;
        const uint32_t v0 = c_t * DEC_TILE + warp * 16, i = v0 + (lane & 15);
        if (i < c_n) {
            const uint32_t j = i < c_sinks ? i : i - c_sinks + c_from, e = p.page.div(j);
            tok = j - e * p.page.d;
            page = p.table[(int64_t)c_b * p.table_row + e];
        }
        next.valid = min(16, max(0, (int)c_n - (int)v0));
        next.b = c_b;
        next.h = c_h;
        next.h0 = c_h0;
        next.t = c_t;
        next.nt = c_nt;
        if (++c_t == c_nt) {
            c_t = 0;
            c_h0 += HEADS;
            if (c_h0 >= p.group) {
                c_h0 = 0;
                if (++c_h == p.hkv && c_left) {
                    c_h = 0;
                    do {
                        ++c_b;
                        visible_keys(p, attn_len(p, c_b), c_sinks, c_from, c_n);
                    } while (c_n == 0);
                    c_nt = (c_n + DEC_TILE - 1) / DEC_TILE;
                }
            }
        }
    };
    const uint32_t ring = sbase + warp * Sh::WARP_STAGE;
    const uint32_t my_row = lane / CPR, my_chunk = lane % CPR;
    const bool in_dim = my_chunk * 8 < p.dim;
    uint32_t to_issue = ntiles;
    // copies of the fetched tile into stage s, then the page numbers of the tile after it
    auto issue = [&](uint32_t s) {
        if (to_issue) {
            --to_issue;
            if (lane == 0) meta[s] = next;
            const uint32_t dst = ring + s * Sh::STAGE;
            // lanes 0 to 15: where the keys lie, lanes 16 to 31: the values
            int64_t off = -1;
            if ((uint32_t)page < p.pages)
                off = lane < 16 ? (int64_t)page * p.k_page + (int64_t)tok * p.k_tok + (int64_t)next.h * p.k_head
                                : (int64_t)page * p.v_page + (int64_t)tok * p.v_tok + (int64_t)next.h * p.v_head;
            else if ((lane & 15) < next.valid) atomicOr(p.status, STATUS_BAD_INDEX);
#pragma unroll
            for (int r = 0; r < 16; r += ROWS_PER) {
                const uint32_t row = r + my_row;
                const uint32_t at = row * ROW + ((my_chunk ^ (row & 7)) << 4);
                const int64_t ko = __shfl_sync(0xFFFFFFFFu, off, row), vo = __shfl_sync(0xFFFFFFFFu, off, 16 + row);
                cp_async16(dst + at, p.k + (ko >= 0 && in_dim ? (ko + my_chunk * 8) * 2 : 0), ko >= 0 && in_dim ? 16 : 0);
                cp_async16(dst + 16 * ROW + at, p.v + (vo >= 0 && in_dim ? (vo + my_chunk * 8) * 2 : 0), vo >= 0 && in_dim ? 16 : 0);
            }
            fetch();
        }
        cp_async_commit();
    };
    fetch();
#pragma unroll
    for (int s = 0; s < STAGES; ++s) issue(s);

    float o[KS][NT][4], m[NT][2], l[NT][2];
    bool fresh = true, begins = true;  // the next tile is the first of an item that this run sees; the run has the item's first tile
    uint32_t s = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < ntiles; ++i) {
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const TileMeta mt = meta[s];
        const uint32_t b = mt.b, h = mt.h, h0 = mt.h0, heads = min((uint32_t)HEADS, p.group - h0);
        if (fresh) {
            fresh = false;
            begins = mt.t == 0;
            // the queries as the B operand, [k step][term][8 heads][lane]; every warp of the CTA has left the previous ones
            for (uint32_t e = threadIdx.x; e < KS * NT * 32; e += DEC_THREADS) {
                const uint32_t ln = e % 32, nt = e / 32 % NT, ks = e / (32 * NT), head = nt * 8 + ln / 4, dim = ks * 16 + 2 * (ln % 4);
                float2 x[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                uint2 raw = make_uint2(0, 0);
                const int64_t at = (int64_t)b * p.q_row + (int64_t)(h * p.group + h0 + head) * p.q_head + dim;
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (head < heads && dim + 8 * j < p.dim) {
                        if constexpr (SPLIT) x[j] = *reinterpret_cast<const float2*>(static_cast<const float*>(p.q) + at + 8 * j);
                        else (j ? raw.y : raw.x) = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.q) + at + 8 * j);
                    }
                if constexpr (!SPLIT) {
                    qf[(ks * NT + nt) * 32 + ln] = raw;
                } else {  // the f32 value as a sum of 16-bit terms, each the rounding of what the ones before left
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        uint2 r;
                        r.x = pack2<F16>(x[0].x, x[0].y);
                        r.y = pack2<F16>(x[1].x, x[1].y);
                        const float2 a = unpack2<F16>(r.x), c = unpack2<F16>(r.y);
                        x[0].x -= a.x, x[0].y -= a.y, x[1].x -= c.x, x[1].y -= c.y;
                        qf[((ks * TERMS + t) * NT + nt) * 32 + ln] = r;
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                m[nt][0] = m[nt][1] = -INFINITY;
                l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[k][nt][c] = 0.f;
            }
        }
        const uint32_t kt = ring + s * Sh::STAGE, vt = kt + 16 * ROW;
        if (mt.valid > 0) {
            // ---- scores: 16 keys x heads
            // partial sums of each term, and of even and odd k steps: products that wait for one another cost more than the adds
            constexpr int CH = NT == 1 && DP <= 128 ? 2 : 1;
            float part[CH * TERMS][NT][4];
#pragma unroll
            for (int c = 0; c < CH * TERMS; ++c)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) part[c][nt][0] = part[c][nt][1] = part[c][nt][2] = part[c][nt][3] = 0.f;
            {
                const uint32_t row = (lane & 7) + (lane & 8);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint32_t a[4];
                    ldsm_x4(a, kt + row * ROW + (((2 * ks + (lane >> 4)) ^ (row & 7)) << 4));
#pragma unroll
                    for (int t = 0; t < TERMS; ++t)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint2 q = qf[((ks * TERMS + t) * NT + nt) * 32 + lane];
                            mma16<F16>(part[CH * t + (ks & (CH - 1))][nt], a, q.x, q.y);
                        }
                }
            }
            float sc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    sc[nt][c] = 0.f;
#pragma unroll
                    for (int t = CH * TERMS - 1; t >= 0; --t) sc[nt][c] += part[t][nt][c];  // the smallest terms first
                }
            // ---- softmax: element c of a lane is key lane / 4 + 8 (c / 2), head 2 (lane % 4) + c % 2 of its eight
            const bool in0 = (lane >> 2) < mt.valid, in1 = (lane >> 2) + 8 < mt.valid;
            float alpha[NT][2];
            uint32_t pt[TERMS][NT][2];  // the weights as a sum of 16-bit terms, too
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float x[4];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float mx = fmaxf(in0 ? sc[nt][c] * p.scale_log2 : -INFINITY, in1 ? sc[nt][c + 2] * p.scale_log2 : -INFINITY);
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
                    mx = fmaxf(mx, m[nt][c]);
                    alpha[nt][c] = mx == -INFINITY ? 1.f : exp2_approx(m[nt][c] - mx);
                    m[nt][c] = mx;
                    const float base = mx == -INFINITY ? 0.f : mx - WEIGHT_BIAS<F16>;
                    x[c] = in0 ? exp2_approx(fmaf(sc[nt][c], p.scale_log2, -base)) : 0.f;
                    x[c + 2] = in1 ? exp2_approx(fmaf(sc[nt][c + 2], p.scale_log2, -base)) : 0.f;
                    l[nt][c] = fmaf(l[nt][c], alpha[nt][c], x[c] + x[c + 2]);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        const uint32_t r = pack2<F16>(x[2 * j], x[2 * j + 1]);
                        pt[t][nt][j] = transpose8(r);
                        if constexpr (TERMS > 1) {
                            const float2 a = unpack2<F16>(r);
                            x[2 * j] -= a.x, x[2 * j + 1] -= a.y;
                        }
                    }
                }
                if constexpr (!SPLIT) {
                    if (__any_sync(0xFFFFFFFFu, alpha[nt][0] != 1.f || alpha[nt][1] != 1.f)) {
#pragma unroll
                        for (int k = 0; k < KS; ++k)
#pragma unroll
                            for (int c = 0; c < 4; ++c) o[k][nt][c] *= alpha[nt][c & 1];
                    }
                }
            }
            // ---- values: 16 elements of the head x heads, over the 16 keys
            const uint32_t key = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t a[4];
                ldsm_x4_t(a, vt + key * ROW + (((2 * k + ((lane >> 3) & 1)) ^ (key & 7)) << 4));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if constexpr (!SPLIT) {
                        mma16<F16>(o[k][nt], a, pt[0][nt][0], pt[0][nt][1]);
                    } else {
                        // the tensor core cuts its sums off: over a long row that would show in an f32 result, so a tile is summed by
                        // itself, smallest terms first, and added with rounding
                        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int t = TERMS - 1; t >= 0; --t) mma16<F16>(x, a, pt[t][nt][0], pt[t][nt][1]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[k][nt][c] = fmaf(o[k][nt][c], alpha[nt][c & 1], x[c]);
                    }
                }
            }
        }
        if (mt.t + 1 == mt.nt || i + 1 == ntiles) {
            // ---- the item, or this run's part of it, is done: join the four warps
            fresh = true;
            const bool whole = begins && mt.t + 1 == mt.nt;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    l[nt][c] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][c], 4);
                    l[nt][c] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][c], 8);
                    l[nt][c] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][c], 16);
                    if (lane < 4) ml[warp * HEADS + nt * 8 + 2 * lane + c] = make_float2(m[nt][c], l[nt][c]);
                }
            __syncthreads();
            // a warp's sums go to its part of the stage that it has just read, [head][DP], groups of eight elements swapped by head
            // so that neither the writes nor the reads of a warp meet in a bank
            float* mine = reinterpret_cast<float*>(smem + warp * Sh::WARP_STAGE + s * Sh::STAGE);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t head = nt * 8 + 2 * (lane & 3) + c;
                    float mx = -INFINITY;
#pragma unroll
                    for (int w = 0; w < DEC_WARPS; ++w) mx = fmaxf(mx, ml[w * HEADS + head].x);
                    const float f = m[nt][c] == -INFINITY ? 0.f : exp2_approx(m[nt][c] - mx);
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int j = 0; j < 2; ++j) mine[head * DP + ((k * 16 + j * 8 + (lane >> 2)) ^ ((lane & 3) << 3))] = o[k][nt][2 * j + c] * f;
                }
            __syncthreads();
            // the part of an item that begins before this run is the run's first, the part of one that ends behind it its last
            float* part = d.part + (size_t)(2 * blockIdx.x + (begins ? 1 : 0)) * Sh::PART;
            for (uint32_t e = threadIdx.x; e < heads * (DP / 4); e += DEC_THREADS) {
                const uint32_t head = e / (DP / 4), dim = 4 * (e % (DP / 4));
                const uint8_t* from = smem + s * Sh::STAGE + 4 * (head * DP + (dim ^ (((head >> 1) & 3) << 3)));
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                float mx = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < DEC_WARPS; ++w) mx = fmaxf(mx, ml[w * HEADS + head].x);
#pragma unroll
                for (int w = 0; w < DEC_WARPS; ++w) {
                    const float4 x = *reinterpret_cast<const float4*>(from + w * Sh::WARP_STAGE);
                    const float2 y = ml[w * HEADS + head];
                    a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
                    if (y.x != -INFINITY) sum = fmaf(y.y, exp2_approx(y.x - mx), sum);
                }
                if (whole) {
                    write_row<F16>(p, b, h * p.group + h0 + head, dim, a, mx, sum);
                } else {
                    *reinterpret_cast<float4*>(part + head * DP + dim) = a;
                    if (dim == 0) part[HEADS * DP + head] = mx, part[HEADS * DP + HEADS + head] = sum;
                }
            }
            if (!whole) {
                // CTAs first .. last share the item; the one whose count completes theirs adds the parts in their order
                const uint64_t g0 = begin + i - mt.t, g1 = g0 + mt.nt - 1;
                const uint32_t first = (uint32_t)(((g0 + 1) * active - 1) / total), last = (uint32_t)(((g1 + 1) * active - 1) / total);
                __threadfence();
                __syncthreads();
                if (threadIdx.x == 0) s_last = atomicAdd(d.counters + first, 1u) == last - first ? 1u : 0u;
                __syncthreads();
                if (s_last) {
                    __threadfence();
                    if (threadIdx.x == 0) d.counters[first] = 0;  // for the next call
                    for (uint32_t e = threadIdx.x; e < heads * (DP / 4); e += DEC_THREADS) {
                        const uint32_t head = e / (DP / 4), dim = 4 * (e % (DP / 4));
                        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                        float mx = -INFINITY, sum = 0.f;
                        constexpr int AT_ONCE = 8;
                        for (uint32_t c0 = first; c0 <= last; c0 += AT_ONCE) {
                            float4 x[AT_ONCE];
                            float pm[AT_ONCE], ps[AT_ONCE], top = mx;
#pragma unroll
                            for (int u = 0; u < AT_ONCE; ++u) {
                                pm[u] = -INFINITY;
                                if (c0 + u <= last) {
                                    const float* q = d.part + (size_t)(2 * (c0 + u) + (c0 + u == first ? 1 : 0)) * Sh::PART;
                                    x[u] = __ldcg(reinterpret_cast<const float4*>(q + head * DP + dim));
                                    pm[u] = __ldcg(q + HEADS * DP + head);
                                    ps[u] = __ldcg(q + HEADS * DP + HEADS + head);
                                }
                            }
#pragma unroll
                            for (int u = 0; u < AT_ONCE; ++u) top = fmaxf(top, pm[u]);
                            const float f0 = mx == -INFINITY ? 0.f : exp2_approx(mx - top);
                            a.x *= f0, a.y *= f0, a.z *= f0, a.w *= f0, sum *= f0;
                            mx = top;
#pragma unroll
                            for (int u = 0; u < AT_ONCE; ++u)
                                if (c0 + u <= last) {
                                    const float f = pm[u] == -INFINITY ? 0.f : exp2_approx(pm[u] - top);
                                    a.x = fmaf(x[u].x, f, a.x), a.y = fmaf(x[u].y, f, a.y), a.z = fmaf(x[u].z, f, a.z), a.w = fmaf(x[u].w, f, a.w);
                                    sum = fmaf(ps[u], f, sum);
                                }
                        }
                        write_row<F16>(p, b, h * p.group + h0 + head, dim, a, mx, sum);
                    }
                }
            }
            __syncthreads();  // the stage, ml and s_last are free again
        }
        __syncwarp();
        issue(s);
        s = s + 1 == STAGES ? 0 : s + 1;
    }
}

template <int DP, int NT, bool F16, bool SPLIT>
cudaError_t decode_go(const AttnParams& p, DecodePlan& d, uint32_t grid, cudaStream_t st) {
    using Sh = DecodeShape<DP, NT, F16, SPLIT>;
    constexpr int MINB = DP == 64 ? 3 : DP == 128 ? 2 : 1;
    auto kernel = decode_kernel<DP, NT, F16, SPLIT, MINB>;
    static PerDeviceOnce once;
    cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM); });
    if (e != cudaSuccess) return e;
    note_launch();
    return launch_pdl(kernel, dim3(grid), dim3(DEC_THREADS), Sh::SMEM, st, p, d);
}
template <int DP, int NT>
cudaError_t decode_typed(const AttnParams& p, DecodePlan& d, uint32_t grid, cudaStream_t st) {
    const bool split = p.q_dtype == DT_F32;
    return p.f16 ? (split ? decode_go<DP, NT, true, true>(p, d, grid, st) : decode_go<DP, NT, true, false>(p, d, grid, st))
                 : (split ? decode_go<DP, NT, false, true>(p, d, grid, st) : decode_go<DP, NT, false, false>(p, d, grid, st));
}

uint32_t padded_dim(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
uint32_t head_tiles(uint32_t group) { return group > 8 ? 2 : 1; }
uint32_t decode_grid(uint32_t dp, int sm_count) { return (uint32_t)sm_count * (dp == 64 ? 3 : dp == 128 ? 2 : 1); }

}  // namespace

size_t decode_workspace_bytes(uint32_t group, uint32_t dim, int sm_count) {
    const size_t dp = padded_dim(dim), nt = head_tiles(group), grid = decode_grid((uint32_t)dp, sm_count);
    return DEC_COUNTER_BYTES + 2 * grid * 8 * nt * (dp + 2) * sizeof(float);
}

cudaError_t launch_decode(const AttnParams& p, void* ws, int sm_count, cudaStream_t st) {
    const uint32_t dp = padded_dim(p.dim), nt = head_tiles(p.group);
    DecodePlan d;
    d.chunks = (p.group + 8 * nt - 1) / (8 * nt);
    d.items = p.hkv * d.chunks;
    d.min_tiles = 1;
    d.counters = static_cast<uint32_t*>(ws);
    d.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + DEC_COUNTER_BYTES);
    // no more CTAs than tiles there can be
    const uint64_t most = (uint64_t)p.requests * d.items * (((uint64_t)p.width * p.page.d + DEC_TILE - 1) / DEC_TILE);
    uint32_t grid = decode_grid(dp, sm_count);
    if (grid > most) grid = (uint32_t)most;
    if (dp == 64) return nt == 1 ? decode_typed<64, 1>(p, d, grid, st) : decode_typed<64, 2>(p, d, grid, st);
    if (dp == 128) return nt == 1 ? decode_typed<128, 1>(p, d, grid, st) : decode_typed<128, 2>(p, d, grid, st);
    return nt == 1 ? decode_typed<256, 1>(p, d, grid, st) : decode_typed<256, 2>(p, d, grid, st);
}

}  // namespace b200q
