// sm_100a attention over the 8-bit paged KV cache (format: cache8.cuh).
//
// out_i = sum_j p_ij v_j / sum_j p_ij, p_ij = 2^(s_ij - m_i), s_ij = scale log2(e) q_i . k_j
// over the tokens j that row i sees, in one pass with the running maximum m. Codes
// meet queries and weights as fp16 (e4m3 is exact in it) in matrix instructions
// with 32-bit sums; a page's key scale multiplies its scores, its value scale its
// weights, both in 32 bits.
#include <mutex>
#include <set>
#include <type_traits>
#include <utility>

#include "cache8.cuh"

namespace {

struct AttendArgs {
    Cache c;
    Batch b;
    Rows query;
    char* out;
    int q_heads, group;       // query heads; query heads a KV head
    float scale;              // of the scores, times log2(e)
    uint32_t* status;
};

// A sequence as the attention kernels see it.
struct Sequence {
    int row, rows, length;    // its token rows, and its tokens with theirs
};

// Reads sequence s; false where it has no rows or does not fit (then recorded).
__device__ __forceinline__ bool read_sequence(const Batch& b, int n, int s, Sequence& q, uint32_t* status) {
    const int from = ints(b.start)[s], to = ints(b.start)[s + 1];
    if (from >= to) return false;
    q.row = from, q.rows = to - from, q.length = ints(b.lengths)[s];
    if (from < 0 || to > b.rows || q.rows > b.max_query || int64_t(q.length) > int64_t(b.width) * n) {
        atomicOr(status, KVSNAP_C8_BAD_LENGTH);
        return false;
    }
    q.length = max(q.length, 0);
    return true;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t half2_of_codes(uint16_t codes) {
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(codes));
    return d;
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
}

// ---- few rows: decode -------------------------------------------------------------------
//
// Sequences with at most kStepRows rows a KV head (query heads of the group times
// new tokens). Bound by the cache's bytes, so nothing but a page's codes is read,
// once, straight into the registers of the lanes whose matrix fragments they are:
// with the keys as the 16-row operand of m16n8k16, lane (g, t) needs 16 bytes of
// tokens' rows g, and with the values' transpose, 16 dims of 4 tokens. Which token
// is row g and which dim is row g of the transpose is free as long as both
// products agree, so it is chosen to make every load a 16-byte one and every pair
// of codes that a fragment register holds adjacent after one byte permute. The
// scores come out transposed, [token][row], and one 8x8 transpose in registers
// makes them the weights' fragment.

constexpr int kStepRows = 16;
constexpr int kWarps = 16;                 // a CTA: HC heads x TS slices of a chunk
constexpr int kGranule = 16;               // tokens a warp takes at a time
constexpr float kLowest = -3e38f;          // the running maximum before any token
constexpr float kSlack = 8.0f;             // log2 by which a weight may exceed 1 before sums are rescaled

struct StepArgs {
    AttendArgs a;
    int hc, ts, hg;           // heads a CTA, slices of a chunk, groups of heads
    float* part;              // [2 * CTAs][hc][rows][D] unfinished sums of units that CTAs share
    float2* part_ml;          // their maxima and weights' sums
    int4* shared_units;       // a CTA: the unit whose first part it holds: first row, head group, rows, parts
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

__device__ __forceinline__ uint4 load16(const char* at) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
    return v;
}

__device__ __forceinline__ uint2 load8bytes(const char* at) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(at));
    return v;
}

// Chunks of a sequence: TS granules each; a sequence without tokens has one, whose rows become zeros.
__device__ __forceinline__ int chunks_of(const StepArgs& p, int s, Sequence& q) {
    if (!read_sequence(p.a.b, p.a.c.block_size, s, q, p.a.status) || q.rows * p.a.group > kStepRows) return 0;
    return max(1, (q.length + p.ts * kGranule - 1) / (p.ts * kGranule));
}

__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* scratch) {
#pragma unroll
    for (int k = 16; k; k >>= 1) v += __shfl_xor_sync(~0u, v, k);
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < int(blockDim.x) / 32; ++w) v += scratch[w];
    __syncthreads();
    return v;
}

// One warp's share of chunks [c0, c1) of one head of one sequence.
template <typename T, int D, int NT>
struct StepWarp {
    static constexpr int kHalves = D / 64, kTiles = D / 16;
    float o[NT][kTiles][4];                // (dim pair, row) sums, relative to m and vref
    float m[NT][2], l[NT][2];              // of rows 8 nt + 2 t, + 1
    float vref;                            // largest value scale so far

    __device__ __forceinline__ void run(const StepArgs& p, const Sequence& q, int s, int head, int slice, int c0,
                                        int c1) {
        const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
        const Cache& c = p.a.c;
        const int rows = q.rows * p.a.group, first_seen = q.length - q.rows + 1;
        vref = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = kLowest, l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int mt = 0; mt < kTiles; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][mt][i] = 0.0f;
        }

        // Queries as fp16, each row times a power of two that brings its largest element to
        // [2^14, 2^15): bf16's exponents do not fit fp16, and what then falls below fp16's
        // normal numbers is under 2^-28 of the row's largest.
        uint32_t qb[NT][kHalves * 4][2];
        float factor[NT][2];               // of rows 8 nt + 2 t, + 1: scores' factor
        int seen[NT][2];                   // tokens that those rows see
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + g;
            float v[kHalves][16], top = 0.0f;
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
                if (r < rows) {
                    const char* at = p.a.query.at + int64_t(q.row + r / p.a.group) * p.a.query.token +
                                     int64_t(head * p.a.group + r % p.a.group) * p.a.query.head + 128 * half + 32 * t;
                    float w[8];
                    load8<T>(at, w);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[half][i] = w[i];
                    load8<T>(at + 16, w);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[half][8 + i] = w[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[half][i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, finite_size(v[half][i]));
            }
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
            const int e = max(int(__float_as_uint(top) >> 23), 27);          // biased
            const float up = __uint_as_float(uint32_t(127 + 14 + 127 - e) << 23);
            const float down = __uint_as_float(uint32_t(max(e - 14, 1)) << 23) * p.a.scale;
#pragma unroll
            for (int half = 0; half < kHalves; ++half)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    qb[nt][half * 4 + w][0] = pack_half2(v[half][4 * w] * up, v[half][4 * w + 1] * up);
                    qb[nt][half * 4 + w][1] = pack_half2(v[half][4 * w + 2] * up, v[half][4 * w + 3] * up);
                }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                factor[nt][i] = __shfl_sync(~0u, down, (2 * t + i) * 4);
                seen[nt][i] = first_seen + (nt * 8 + 2 * t + i) / p.a.group;
            }
        }

        const int token_a = 4 * (g >> 1) + (g & 1);                            // of score row g; row g + 8: + 2
        const char* keys = reinterpret_cast<const char*>(c.codes) + head * c.head_pitch;
        const char* k_lane = keys + token_a * c.token_pitch + 16 * t;
        const char* v_lane = keys + c.side_pitch + 4 * t * c.token_pitch + (D / 8) * g;
        const int64_t two_tokens = 2 * c.token_pitch;

        uint4 kr[kHalves][2], vr[4];
        const auto load_keys = [&](int64_t off) {
#pragma unroll
            for (int half = 0; half < kHalves; ++half)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    kr[half][i] = off >= 0 ? load16(k_lane + off + i * two_tokens + 64 * half) : make_uint4(0, 0, 0, 0);
        };
        const auto load_values = [&](int64_t off) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                vr[j] = make_uint4(0, 0, 0, 0);
                if (off >= 0) {
                    if constexpr (D == 128) {
                        vr[j] = load16(v_lane + off + j * c.token_pitch);
                    } else {
                        const uint2 x = load8bytes(v_lane + off + j * c.token_pitch);
                        vr[j].x = x.x, vr[j].y = x.y;
                    }
                }
            }
        };

        // Pages of 32 chunks at a time, one a lane: where the warp's granule lies, and its scales.
        int64_t off = -1;
        float ks = 0.0f, vs = 0.0f;
        const auto look_up = [&](int chunk) {
            const int64_t token = (int64_t(chunk + lane) * p.ts + slice) * kGranule;
            off = -1, ks = vs = 0.0f;
            if (chunk + lane < c1 && token < q.length) {
                const int64_t block = ints(p.a.b.table)[s * p.a.b.table_pitch + token / c.block_size];
                if (block < 0 || block >= c.blocks) {
                    atomicOr(p.a.status, KVSNAP_DP_BAD_BLOCK);
                } else {
                    off = block * c.block_pitch + token % c.block_size * c.token_pitch;
                    const float* scales = reinterpret_cast<const float*>(c.scales) + block * 2 * c.kv_heads + head;
                    ks = scales[0], vs = scales[c.kv_heads];
                }
            }
        };

        look_up(c0);
        int64_t now = __shfl_sync(~0u, off, 0);
        load_keys(now);
        load_values(now);
        for (int chunk = c0; chunk < c1; ++chunk) {
            const int j = (chunk - c0) % 32;
            const float k_scale = __shfl_sync(~0u, ks, j), v_scale = __shfl_sync(~0u, vs, j);
            const bool dead = now < 0;
            if (j == 31) look_up(chunk + 1);
            const int64_t next = __shfl_sync(~0u, off, (j + 1) % 32);
            const int64_t base = (int64_t(chunk) * p.ts + slice) * kGranule;

            float sc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
                const uint32_t wa[4] = {kr[half][0].x, kr[half][0].y, kr[half][0].z, kr[half][0].w};
                const uint32_t wb[4] = {kr[half][1].x, kr[half][1].y, kr[half][1].z, kr[half][1].w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t a0 = half2_of_codes(uint16_t(wa[w])), a2 = half2_of_codes(uint16_t(wa[w] >> 16));
                    const uint32_t a1 = half2_of_codes(uint16_t(wb[w])), a3 = half2_of_codes(uint16_t(wb[w] >> 16));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma16816(sc[nt], a0, a1, a2, a3, qb[nt][half * 4 + w][0], qb[nt][half * 4 + w][1]);
                }
            }
            load_keys(next);

            // Edge: tokens that some row does not see, or a page that is not there.
            const bool edge = dead || base + kGranule > first_seen;
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float f = factor[nt][i] * k_scale;
                    sc[nt][i] *= f, sc[nt][2 + i] *= f;
                    if (edge) {
                        if (dead || base + token_a >= seen[nt][i]) sc[nt][i] = -INFINITY;
                        if (dead || base + token_a + 2 >= seen[nt][i]) sc[nt][2 + i] = -INFINITY;
                    }
                    grow |= fmaxf(sc[nt][i], sc[nt][2 + i]) > m[nt][i] + kSlack;
                }
            }
            if (__any_sync(~0u, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float top = fmaxf(sc[nt][i], sc[nt][2 + i]);
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
                        top = fmaxf(top, m[nt][i]);
                        const float keep = exp2_fast(m[nt][i] - top);
                        m[nt][i] = top, l[nt][i] *= keep;
#pragma unroll
                        for (int mt = 0; mt < kTiles; ++mt) o[nt][mt][i] *= keep, o[nt][mt][2 + i] *= keep;
                    }
            }
            // Weights carry the page's value scale relative to the largest so far, so fp16 holds them.
            if (v_scale > vref) {
                const float keep = vref / v_scale;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int mt = 0; mt < kTiles; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[nt][mt][i] *= keep;
                vref = v_scale;
            }
            const float part = vref > 0.0f ? v_scale / vref : 0.0f;
            uint32_t pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = exp2_fast(sc[nt][i] - m[nt][i % 2]);
                l[nt][0] += w[0] + w[2], l[nt][1] += w[1] + w[3];
                pb[nt][0] = transpose8x8(pack_half2(w[0] * part, w[1] * part));
                pb[nt][1] = transpose8x8(pack_half2(w[2] * part, w[3] * part));
            }

            const auto add_values = [&](const uint4 (&v)[4], const uint32_t (&b)[NT][2]) {
                const uint32_t w[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w}, {v[1].x, v[1].y, v[1].z, v[1].w},
                                          {v[2].x, v[2].y, v[2].z, v[2].w}, {v[3].x, v[3].y, v[3].z, v[3].w}};
#pragma unroll
                for (int mt = 0; mt < kTiles; ++mt) {
                    const uint32_t pick = mt % 2 ? 0x7362 : 0x5140;
                    const uint32_t x = __byte_perm(w[0][mt / 2], w[1][mt / 2], pick);
                    const uint32_t y = __byte_perm(w[2][mt / 2], w[3][mt / 2], pick);
                    const uint32_t a0 = half2_of_codes(uint16_t(x)), a1 = half2_of_codes(uint16_t(x >> 16));
                    const uint32_t a2 = half2_of_codes(uint16_t(y)), a3 = half2_of_codes(uint16_t(y >> 16));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][mt], a0, a1, a2, a3, b[nt][0], b[nt][1]);
                }
            };
            if (!edge) {
                add_values(vr, pb);
            } else if (!dead) {
                // One new token at a time, with the values it does not see left out: a weight of 0
                // times what a masked slot holds (NaN, say) must not reach it.
                for (int i = 0; i < q.rows; ++i) {
                    if (first_seen + i <= base) continue;
                    uint4 v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        v[k] = base + 4 * t + k < first_seen + i ? vr[k] : make_uint4(0, 0, 0, 0);
                    uint32_t b[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int k = 0; k < 2; ++k) b[nt][k] = (nt * 8 + g) / p.a.group == i ? pb[nt][k] : 0u;
                    add_values(v, b);
                }
            }
            load_values(next);
            now = next;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], 4);
                l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], 8);
                l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], 16);
            }
    }
};

template <int D, int NT>
struct StepShared {
    static constexpr int kPitch = D + 4;
    float o[kWarps][8 * NT][kPitch];
    float2 ml[kWarps][8 * NT];
    int64_t scratch[kWarps];
    int64_t prefix[kWarps];
    int64_t found_first;
    int found;
};

// 4 outputs of a row.
template <typename T>
__device__ __forceinline__ void store4(char* at, float4 v) {
    *reinterpret_cast<uint2*>(at) = make_uint2(T::pack(v.x, v.y), T::pack(v.z, v.w));
}

// SPLIT: the chunks of all sequences and head groups, end to end, are cut evenly over the CTAs; units
// (a sequence's head group) that CTAs share leave parts in the workspace. Otherwise CTA i is unit i.
template <typename T, int D, int NT, bool SPLIT>
__global__ void __launch_bounds__(32 * kWarps, 1) step_kernel(const __grid_constant__ StepArgs p) {
    extern __shared__ char raw[];
    auto& sh = *reinterpret_cast<StepShared<D, NT>*>(raw);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, seqs = p.a.b.seqs;
    asm volatile("griddepcontrol.launch_dependents;");

    int64_t total = 0, ctas = 0, pos = 0, end = 0;
    int s = 0, hg = 0, c0 = 0;
    Sequence q;
    if (SPLIT) {
        if (threadIdx.x == 0) p.shared_units[blockIdx.x] = make_int4(0, 0, 0, 0);
        int64_t mine = 0;
        for (int i = threadIdx.x; i < seqs; i += blockDim.x) mine += int64_t(chunks_of(p, i, q)) * p.hg;
        total = block_sum(mine, sh.scratch);
        ctas = min(int64_t(gridDim.x), total);                     // that have work: a chunk at least
        if (blockIdx.x >= ctas) return;
        pos = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
        // The sequence that chunk `pos` lies in, and the chunk at which it begins.
        int64_t before = 0;
        for (int tile = 0; tile < seqs; tile += blockDim.x) {
            const int i = tile + threadIdx.x;
            const int64_t n = i < seqs ? int64_t(chunks_of(p, i, q)) * p.hg : 0;
            int64_t sum = n;
#pragma unroll
            for (int k = 1; k < 32; k <<= 1) {
                const int64_t up = __shfl_up_sync(~0u, sum, k);
                if (lane >= k) sum += up;
            }
            if (lane == 31) sh.prefix[warp] = sum;
            __syncthreads();
            int64_t all = 0, low = before;
            for (int w = 0; w < kWarps; ++w) {
                if (w == warp) low = before + all;
                all += sh.prefix[w];
            }
            const int64_t first = low + sum - n;
            if (n && first <= pos && pos < first + n) sh.found = i, sh.found_first = first;
            before += all;
            __syncthreads();
            if (before > pos) break;
        }
        s = sh.found;
        const int n = chunks_of(p, s, q);
        hg = int((pos - sh.found_first) / n), c0 = int((pos - sh.found_first) % n);
    } else {
        s = blockIdx.x / p.hg, hg = blockIdx.x % p.hg;
        end = 1;
    }

    while (pos < end && s < seqs) {
        const int chunks = chunks_of(p, s, q);
        if (!chunks) {
            if (!SPLIT) return;
            ++s;
            continue;
        }
        const int c1 = SPLIT ? int(min(int64_t(chunks), c0 + (end - pos))) : chunks;
        const int rows = q.rows * p.a.group;
        const int hc = warp % p.hc, slice = warp / p.hc;
        if (slice < p.ts) {
            StepWarp<T, D, NT> w;
            w.run(p, q, s, hg * p.hc + hc, slice, c0, c1);
            const int g = lane / 4, t = lane % 4;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int n = nt * 8 + 2 * t + i;
                    if (g == 0) sh.ml[warp][n] = make_float2(w.m[nt][i], w.l[nt][i]);
#pragma unroll
                    for (int mt = 0; mt < D / 16; mt += 2)
                        *reinterpret_cast<float4*>(&sh.o[warp][n][(D / 8) * g + 2 * mt]) =
                            make_float4(w.o[nt][mt][i] * w.vref, w.o[nt][mt][2 + i] * w.vref,
                                        w.o[nt][mt + 1][i] * w.vref, w.o[nt][mt + 1][2 + i] * w.vref);
                }
            }
        }
        __syncthreads();
        // Join the slices, 4 dims of one row and head a thread.
        const bool whole = !SPLIT || (c0 == 0 && c1 == chunks);
        const int slot = 2 * int(blockIdx.x) + (c0 == 0);
        for (int i = threadIdx.x; i < p.hc * rows * (D / 4); i += blockDim.x) {
            const int at = i % (D / 4) * 4, row = i / (D / 4) % rows, h = i / (D / 4) / rows;
            float top = kLowest;
            for (int k = 0; k < p.ts; ++k) top = fmaxf(top, sh.ml[k * p.hc + h][row].x);
            float sum = 0.0f;
            float4 o = make_float4(0, 0, 0, 0);
            for (int k = 0; k < p.ts; ++k) {
                const float2 ml = sh.ml[k * p.hc + h][row];
                const float f = exp2_fast(ml.x - top);
                const float4 v = *reinterpret_cast<const float4*>(&sh.o[k * p.hc + h][row][at]);
                sum += f * ml.y;
                o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
            }
            const int head = hg * p.hc + h;
            if (whole) {
                // l is 0 only for a row that sees nothing
                const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
                const int64_t to = int64_t(q.row + row / p.a.group) * p.a.q_heads + head * p.a.group + row % p.a.group;
                store4<T>(p.a.out + (to * D + at) * 2, make_float4(o.x * by, o.y * by, o.z * by, o.w * by));
            } else {
                const int64_t to = (int64_t(slot) * p.hc + h) * kStepRows + row;
                *reinterpret_cast<float4*>(p.part + to * D + at) = o;
                if (at == 0) p.part_ml[to] = make_float2(top, sum);
            }
        }
        if (SPLIT) {
            if (!whole && c0 == 0 && threadIdx.x == 0) {
                const int64_t past = pos + chunks;                             // the unit's end
                const int last = int((past * ctas - 1) / total);
                p.shared_units[blockIdx.x] = make_int4(q.row, hg, rows, last - int(blockIdx.x) + 1);
            }
            __syncthreads();
        }
        pos += c1 - c0;
        c0 = 0;
        if (++hg == p.hg) hg = 0, ++s;
    }
}

// Joins the parts of shared units. A unit's parts lie in consecutive CTAs' slots: its first CTA's
// second slot, then first slots. A warp a row where there are few parts, else a CTA a row.
constexpr int kJoinWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ StepArgs p, int ctas) {
    constexpr int kEach = D / 32;
    __shared__ int4 units[512];
    __shared__ int owner[512];
    __shared__ int count, most;
    __shared__ float sums[kJoinWarps][D];
    __shared__ float weight[512], stat[kJoinWarps];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (threadIdx.x == 0) count = most = 0;
    __syncthreads();
    if (warp == 0) {
        int n = 0, parts = 0;
        for (int i = lane; i < (ctas + 31) / 32 * 32; i += 32) {
            const int4 u = i < ctas ? p.shared_units[i] : make_int4(0, 0, 0, 0);
            const uint32_t hit = __ballot_sync(~0u, u.w > 0);
            if (u.w > 0) {
                const int at = n + __popc(hit & ((1u << lane) - 1));
                units[at] = u, owner[at] = i;
                parts = max(parts, u.w);
            }
            n += __popc(hit);
        }
        parts = __reduce_max_sync(~0u, parts);
        if (lane == 0) count = n, most = parts;
    }
    __syncthreads();
    const bool alone = most <= 8;                                  // a warp a row
    const int first = alone ? blockIdx.x * kJoinWarps + warp : blockIdx.x;
    const int step = alone ? gridDim.x * kJoinWarps : gridDim.x;
    for (int task = first; task < count * p.hc * kStepRows; task += step) {
        const int k = task / (p.hc * kStepRows), h = task / kStepRows % p.hc, row = task % kStepRows;
        const int4 u = units[k];
        if (row >= u.z) continue;
        const auto at = [&](int f) -> int64_t {
            return (int64_t(2 * (owner[k] + f) + (f == 0)) * p.hc + h) * kStepRows + row;
        };
        float o[kEach] = {}, sum = 0.0f;
        const auto add = [&](int f, float by) {
            const float* from = p.part + at(f) * D + lane * kEach;
#pragma unroll
            for (int i = 0; i < kEach; ++i) o[i] += by * from[i];
        };
        if (alone) {
            const float2 ml = lane < u.w ? p.part_ml[at(lane)] : make_float2(kLowest, 0.0f);
            float top = ml.x;
#pragma unroll
            for (int i = 4; i; i >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, i));
            top = __shfl_sync(~0u, top, 0);
            const float f = exp2_fast(ml.x - top);
            sum = lane < u.w ? f * ml.y : 0.0f;
#pragma unroll
            for (int i = 4; i; i >>= 1) sum += __shfl_xor_sync(~0u, sum, i);
            sum = __shfl_sync(~0u, sum, 0);
            for (int i = 0; i < u.w; ++i) add(i, __shfl_sync(~0u, f, i));
        } else {
            float top = kLowest;
            for (int i = threadIdx.x; i < u.w; i += blockDim.x) top = fmaxf(top, p.part_ml[at(i)].x);
            top = warp_max(top);
            if (lane == 0) stat[warp] = top;
            __syncthreads();
            top = stat[0];
            for (int w = 1; w < kJoinWarps; ++w) top = fmaxf(top, stat[w]);
            __syncthreads();
            for (int i = threadIdx.x; i < u.w; i += blockDim.x) {
                const float2 ml = p.part_ml[at(i)];
                const float f = exp2_fast(ml.x - top);
                weight[i] = f;
                sum += f * ml.y;
            }
#pragma unroll
            for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(~0u, sum, i);
            if (lane == 0) stat[warp] = sum;
            __syncthreads();
            sum = 0.0f;
            for (int w = 0; w < kJoinWarps; ++w) sum += stat[w];
#pragma unroll 4
            for (int i = warp; i < u.w; i += kJoinWarps) add(i, weight[i]);
#pragma unroll
            for (int i = 0; i < kEach; ++i) sums[warp][lane * kEach + i] = o[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                o[i] = 0.0f;
                for (int w = 0; w < kJoinWarps; ++w) o[i] += sums[w][lane * kEach + i];
            }
            __syncthreads();
            if (warp) continue;
        }
        const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int head = u.y * p.hc + h;
        const int64_t to = int64_t(u.x + row / p.a.group) * p.a.q_heads + head * p.a.group + row % p.a.group;
        char* out = p.a.out + (to * D + lane * kEach) * 2;
        if constexpr (kEach == 4) store4<T>(out, make_float4(o[0] * by, o[1] * by, o[2] * by, o[3] * by));
        else *reinterpret_cast<uint32_t*>(out) = T::pack(o[0] * by, o[1] * by);
    }
}

// One warp: one row and query head, a token at a time with the running maximum and sum.
template <typename T, int D>
__global__ void __launch_bounds__(256) attend_rows_kernel(const __grid_constant__ AttendArgs a) {
    constexpr int kEach = D / 32;
    const int lane = threadIdx.x % 32;
    const int64_t u = int64_t(blockIdx.x) * 8 + threadIdx.x / 32;
    const int64_t row = u / a.q_heads;
    const int head = int(u % a.q_heads), kv = head / (a.q_heads / a.c.kv_heads), n = a.c.block_size;
    if (row >= a.b.rows) return;
    const int32_t* start = ints(a.b.start);
    int lo = 0, hi = a.b.seqs;                       // the first sequence that ends behind the row
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (start[mid + 1] > row) hi = mid; else lo = mid + 1;
    }
    if (lo >= a.b.seqs || row < start[lo]) return;
    if ((start[lo + 1] - start[lo]) * (a.q_heads / a.c.kv_heads) <= kStepRows) return;
    const int to = start[lo + 1], length = ints(a.b.lengths)[lo];
    int64_t seen = length - (to - row) + 1;
    if (to > a.b.rows || to - start[lo] > a.b.max_query || length > int64_t(a.b.width) * n) {
        atomicOr(a.status, KVSNAP_C8_BAD_LENGTH);
        return;
    }
    const uint16_t* q16 = reinterpret_cast<const uint16_t*>(a.query.at + row * a.query.token + head * a.query.head);
    float q[kEach], o[kEach], top = -INFINITY, sum = 0.0f;
    for (int i = 0; i < kEach; ++i) {
        q[i] = T::wide(q16[lane * kEach + i]).x * a.scale;
        o[i] = 0.0f;
    }
    const char* codes = reinterpret_cast<const char*>(a.c.codes);
    const float* scales = reinterpret_cast<const float*>(a.c.scales);
    for (int64_t j = 0; j < seen; ++j) {
        const int64_t block = ints(a.b.table)[lo * a.b.table_pitch + j / n];
        if (block < 0 || block >= a.c.blocks) {
            atomicOr(a.status, KVSNAP_DP_BAD_BLOCK);
            continue;
        }
        const char* k = codes + block * a.c.block_pitch + (j % n) * a.c.token_pitch + kv * a.c.head_pitch + lane * kEach;
        const char* v = k + a.c.side_pitch;
        const float ks = scales[(block * 2) * a.c.kv_heads + kv], vs = scales[(block * 2 + 1) * a.c.kv_heads + kv];
        float s = 0.0f;
        for (int i = 0; i < kEach; ++i) s += q[i] * from_e4m3x2(uint8_t(k[i])).x;
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
        s *= ks;
        const float now = fmaxf(top, s), keep = exp2_fast(top - now), p = exp2_fast(s - now);
        sum = sum * keep + p;
        for (int i = 0; i < kEach; ++i) o[i] = o[i] * keep + p * vs * from_e4m3x2(uint8_t(v[i])).x;
        top = now;
    }
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (row * a.q_heads + head) * D + lane * kEach;
    for (int i = 0; i < kEach; ++i) out[i] = uint16_t(T::pack(sum == 0.0f ? 0.0f : o[i] / sum, 0.0f));
}

// ---- host side ----------------------------------------------------------------------------

// How a call is laid out; the same for its workspace and its launches.
struct StepPlan {
    StepArgs args;
    bool any, split, wide;    // any sequence can be here; units are cut; more than 8 rows a head
    int64_t ctas;
    int64_t part_bytes, ml_bytes, unit_bytes;
};

int sm_count() {
    int device = 0, sms = 0;
    check(cudaGetDevice(&device));
    check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    return sms;
}

StepPlan plan_step(const Cache& c, const Batch& b, int q_heads, int sms) {
    StepPlan plan{};
    StepArgs& p = plan.args;
    const int group = q_heads / c.kv_heads;
    plan.any = group <= kStepRows;
    plan.wide = int64_t(group) * b.max_query > 8;
    for (p.hc = c.kv_heads < 8 ? c.kv_heads : 8; c.kv_heads % p.hc; --p.hc) {}
    p.ts = kWarps / p.hc, p.hg = c.kv_heads / p.hc;
    const int64_t most = (int64_t(b.width) * c.block_size + p.ts * kGranule - 1) / (p.ts * kGranule);
    const int64_t units = int64_t(b.seqs) * p.hg;
    // Up to 8 chunks a unit, a CTA each: cutting them would cost more (a scan of the lengths,
    // parts and their join) than a few granules in turn.
    plan.split = most > 8;
    plan.ctas = plan.split ? sms : units;
    if (plan.split) {
        plan.part_bytes = 2 * plan.ctas * p.hc * kStepRows * c.head_dim * int64_t(sizeof(float));
        plan.ml_bytes = 2 * plan.ctas * p.hc * kStepRows * int64_t(sizeof(float2));
        plan.unit_bytes = plan.ctas * int64_t(sizeof(int4));
    }
    return plan;
}

// Raise a kernel's shared memory limit on the current device, once per kernel and device.
void allow_shared(const void* kernel, int bytes) {
    static std::mutex mu;
    static std::set<std::pair<const void*, int>> done;
    int device = 0;
    check(cudaGetDevice(&device));
    std::lock_guard<std::mutex> hold(mu);
    if (done.count({kernel, device})) return;
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.insert({kernel, device});
}

template <typename K, typename... A>
void launch(K kernel, int64_t ctas, int threads, size_t shared, cudaStream_t stream, bool after, const A&... args) {
    if (shared > 48 << 10) allow_shared(reinterpret_cast<const void*>(kernel), int(shared));
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(unsigned(ctas)), config.blockDim = dim3(unsigned(threads));
    config.dynamicSmemBytes = shared, config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute, config.numAttrs = after ? 1 : 0;
    check(cudaLaunchKernelEx(&config, kernel, args...));
}

template <typename T, int D, int NT>
void launch_step(const StepPlan& plan, cudaStream_t stream) {
    const size_t shared = sizeof(StepShared<D, NT>);
    if (plan.split) launch(step_kernel<T, D, NT, true>, plan.ctas, 32 * kWarps, shared, stream, false, plan.args);
    else launch(step_kernel<T, D, NT, false>, plan.ctas, 32 * kWarps, shared, stream, false, plan.args);
}

void check_attend(const Cache* cache, const Batch* batch, int q_heads) {
    check_cache(cache);
    check_batch(batch);
    require(q_heads > 0 && q_heads % cache->kv_heads == 0, "query heads must be a multiple of the KV heads");
    require(int64_t(batch->seqs) * cache->kv_heads < (1LL << 31), "too many sequences for one attention");
}

}  // namespace

extern "C" int kvsnap_c8_attend_workspace(const kvsnap_c8_cache* cache, const kvsnap_c8_batch* batch, int q_heads,
                                          size_t* bytes) {
    return on_device(cache ? cache->device : 0, [&] {
        check_attend(cache, batch, q_heads);
        *bytes = 0;
        return batch->rows && batch->seqs;
    }, [&] {
        const StepPlan plan = plan_step(*cache, *batch, q_heads, sm_count());
        *bytes = size_t(plan.any ? plan.part_bytes + plan.ml_bytes + plan.unit_bytes : 0);
    });
}

extern "C" int kvsnap_c8_attend(const kvsnap_c8_cache* cache, const kvsnap_c8_batch* batch, int type,
                                const void* query, int64_t query_token, int64_t query_head, int q_heads, float scale,
                                void* out, void* workspace, size_t workspace_bytes, uint32_t* status,
                                uintptr_t stream) {
    return on_device(cache ? cache->device : 0, [&] {
        check_attend(cache, batch, q_heads);
        require(status, "the attention needs a status word");
        if (!batch->rows || !batch->seqs) return false;
        check_rows(query, query_token, query_head);
        require(out, "the attention needs an output");
        require(aligned(reinterpret_cast<intptr_t>(out)), "the output must be 16-byte aligned");
        check_type(type);
        return true;
    }, [&] {
        const AttendArgs a{*cache, *batch, {static_cast<const char*>(query), query_token, query_head},
                           static_cast<char*>(out), q_heads, q_heads / cache->kv_heads, scale * 1.4426950408889634f,
                           status};
        const auto s = reinterpret_cast<cudaStream_t>(stream);
        StepPlan plan = plan_step(*cache, *batch, q_heads, sm_count());
        const int64_t needed = plan.any ? plan.part_bytes + plan.ml_bytes + plan.unit_bytes : 0;
        require(!needed || (workspace && int64_t(workspace_bytes) >= needed &&
                            aligned(reinterpret_cast<intptr_t>(workspace))),
                "the attention's workspace is too small or not 16-byte aligned");
        plan.args.a = a;
        plan.args.part = static_cast<float*>(workspace);
        plan.args.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + plan.part_bytes);
        plan.args.shared_units =
            reinterpret_cast<int4*>(static_cast<char*>(workspace) + plan.part_bytes + plan.ml_bytes);
        by_type(type, cache->head_dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int D = decltype(d)::value;
            if (plan.any) {
                if (plan.wide) launch_step<T, D, 2>(plan, s);
                else launch_step<T, D, 1>(plan, s);
                if (plan.split)
                    launch(join_kernel<T, D>, plan.ctas, 32 * kJoinWarps, 0, s, true, plan.args, int(plan.ctas));
            }
            if (int64_t(a.group) * batch->max_query > kStepRows)
                attend_rows_kernel<T, D><<<unsigned((int64_t(batch->rows) * q_heads + 7) / 8), 256, 0, s>>>(a);
        });
        check(cudaGetLastError());
    });
}
