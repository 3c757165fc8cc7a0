// sm_100a attention over the 8-bit paged KV cache (format: cache8.cuh).
//
// out_i = sum_j p_ij v_j / sum_j p_ij, p_ij = 2^(s_ij - m_i), s_ij = scale log2(e) q_i . k_j
// over the tokens j that row i sees, in one pass with the running maximum m. Codes
// meet queries and weights as fp16 (e4m3 is exact in it) in matrix instructions
// with 32-bit sums; a page's key scale multiplies its scores, its value scale its
// weights, both in 32 bits. Weights meet values as fp16, so they are held relative to a
// second running maximum, of weight times value scale: a page of large values and next to
// no weight then takes no bits from the pages that make up the result.
#include <type_traits>

#include "cache8.cuh"

namespace {

struct AttendArgs {
    Cache c;
    Batch b;
    Rows query;
    char* out;
    int q_heads, group;       // query heads; query heads a KV head
    int step_rows;            // sequences of up to so many rows a KV head are the step kernel's
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

// Four codes as two pairs of fp16, exactly.
__device__ __forceinline__ void halves_of_codes(uint32_t codes, uint32_t& low, uint32_t& high) {
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(low), "=r"(high) : "r"(codes));
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
}

// A kernel's work is cut evenly over its CTAs, so neighbours share units (a sequence's head, or group of
// heads, and a tile of its rows). A CTA that holds a part of one leaves the part's sums here: in its
// second slot where the part begins the unit, in its first where it goes on with one.
struct SharedUnit {
    int row;                  // the sequence's first token row
    int head;                 // first KV head
    int first, rows;          // rows [first, first + rows) of each head (row r: token r / group, head r % group)
    int parts;                // CTAs that share it, from this one on; 0: none
};

// Work of `total`, cut evenly over at most `most` CTAs (a piece of at least 1 each).
struct Cut {
    uint32_t ctas, each, more;     // pieces of each + 1, then of each

    __device__ __forceinline__ Cut(uint32_t total, uint32_t most) : ctas(min(total, most)) {
        each = ctas ? total / ctas : 0, more = ctas ? total % ctas : 0;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t cta) const { return cta * each + min(cta, more); }
    // The CTA that place `at` is of.
    __device__ __forceinline__ uint32_t of(uint32_t at) const {
        const uint32_t long_ones = more * (each + 1);
        return at < long_ones ? at / (each + 1) : more + (at - long_ones) / each;
    }
};

struct Parts {
    float* sums;              // [2 * CTAs][slot rows][D]
    float2* ml;               // their maxima and weights' sums
    SharedUnit* units;        // a CTA's unit that it begins and others go on with
    int heads, head_rows;     // slot rows: heads x rows a head
    int used_rows;            // that a head can have in this call
};

// ---- few rows: decode -------------------------------------------------------------------
//
// Sequences with at most kStepRows rows a KV head (query heads of the group times
// new tokens): what m16n8k16 products take without idle rows, while the kernel below works on 256 rows
// whatever there are (16 sequences of 8000 tokens with 8 rows a head: 58 us, there 153; with 16 rows, whose
// registers spill at 128 dims, 98; 64 of 512 to 8192 with 4, 8, 16 and 24 rows 107, 110, 185 and, there, 323).
// Bound by the cache's bytes, so nothing but a page's codes is read, once: a step of 64 sessions of 512 to
// 8192 tokens with 8 heads of 128, 372 MB, takes 70 us, 5.3 TB/s, of which the loop over granules runs at 86 %
// of the rate of a plain copy, and the rest is the scan for a CTA's chunks (2 us), the first copies'
// way and the merge of a CTA's slices (2 us a unit). With few sequences those are what bounds it: 21 us for
// one of 32k tokens, whose 67 MB are 10 us. A warp copies a granule of 16 tokens to its own shared memory
// asynchronously, kAhead granules ahead, no warp waiting for another; 8 lanes copy
// one token's line, as 16-byte requests are joined among 8 lanes (with lanes that
// each fetched the codes of their own fragments, 32 bytes of a line a request, this
// kernel reached 4.1 TB/s). With the keys as the 16-row operand of m16n8k16 a
// lane (g, t) then needs 16 bytes of tokens' rows g, and with the values'
// transpose, 16 dims of 4 tokens. Which token is row g and which dim is row g of
// the transpose is free as long as both products agree, so it is chosen to make
// every read a 16-byte one and every pair of codes that a fragment register holds
// adjacent after one byte permute. The scores come out transposed, [token][row],
// and one 8x8 transpose in registers makes them the weights' fragment.

constexpr int kStepRows = 16;
constexpr int kWarps = 16;                 // a CTA: HC heads x TS slices of a chunk
// What a unit costs besides its chunks (its first pages and copies, which wait for the unit before, and its
// merge), in chunks: work is cut by chunks and this. Without it, with 3, 5, 9 (us): a 32k step of 64 and 8
// heads 31.0, 27.7, 25.8, 25.4; 16 sequences of up to 32k tokens of one head 29.4, 25.6, 23.8, 23.7; 64
// sessions of 1k to 8k 94.5, 90.0, 89.3, 91.0; 16 of mixed rows 65.3, 59.5, 60.7, 64.8.
constexpr int kStepUnitCost = 5;
constexpr int kSpread = 48;                // units of few sequences that heads are spread for
constexpr int kAhead = 3;                  // granules a warp holds: one in use, the others on their way
constexpr float kLowest = -1e38f;          // the running maxima before any token
constexpr float kSlack = 14.0f;            // log2 by which a weight may exceed 1 before sums are rescaled (fp16: 2^16)

struct StepArgs {
    AttendArgs a;
    int hc, ts, hg;           // heads a CTA, slices of a chunk, groups of heads
    Parts parts;
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

// 16 bytes of a cache that are read once, or zeros. Predicated, not branched around: where a branch
// around a load joins, the load is waited for.
__device__ __forceinline__ uint4 load16(const char* at, bool there) {
    uint4 v;
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %5, 0;\nmov.u32 %0, 0;\nmov.u32 %1, 0;\nmov.u32 %2, 0;\nmov.u32 %3, 0;\n"
                 "@p ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n}"
                 : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(at), "r"(uint32_t(there)));
    return v;
}

// 16 bytes to shared memory, or zeros, on their way until copies_done.
__device__ __forceinline__ void copy_async(uint32_t to, const char* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

__device__ __forceinline__ void copy_async4(uint32_t to, const float* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

// Where 16 bytes `chunk` of a token's D codes lie in a granule of one side: lines of 128 bytes, their 16-byte
// places turned so that the 8 lanes of a read meet all banks. Such lanes read the keys of tokens 4 k and
// 4 k + 1 (+ 2), and 2 chunks of the values of tokens i, 4 + i, 8 + i, 12 + i.
template <int D, bool VALUES>
__device__ __forceinline__ uint32_t in_granule(int token, int chunk) {
    const int line = token * D / 128, place = token * D % 128 / 16 + chunk;
    return uint32_t(line * 128 + (place ^ (VALUES ? token / 4 * 2 : D == 128 ? token % 2 * 4 : 0)) * 16);
}

// All of the thread's copies but its last n groups.
template <int N>
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void copies_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }

__device__ __forceinline__ uint2 read_shared8(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ uint4 read_shared(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// A scale as 2^power * part, part in [1, 2): the weights of its values take the power into their exponent.
// Of a scale of 0 the part is 0 and the power -infinity, which raises no maximum.
struct ValueScale {
    float power, part;

    __device__ __forceinline__ explicit ValueScale(float s) {
        const int bits = min(max(int(__float_as_uint(s) >> 23), 1), 253);
        part = s * __uint_as_float(uint32_t(254 - bits) << 23);
        power = part > 0.0f ? float(bits - 127) : -INFINITY;
    }
};

// Where a warp's granule of a chunk lies, and its scales. A page that is not there: off < 0.
struct __align__(16) StepPage {
    int64_t off;
    float ks, vs;
};

// Chunks of a sequence: TS granules each; a sequence without tokens has one, whose rows become zeros.
__device__ __forceinline__ int chunks_of(const StepArgs& p, int s, Sequence& q) {
    if (!read_sequence(p.a.b, p.a.c.block_size, s, q, p.a.status) || q.rows * p.a.group > p.a.step_rows) return 0;
    return max(1, (q.length + p.ts * kGranule - 1) / (p.ts * kGranule));
}

// What a head group of a sequence costs: its chunks, and what it costs besides; without chunks nothing.
__device__ __forceinline__ int cost_of(const StepArgs& p, int s, Sequence& q) {
    const int chunks = chunks_of(p, s, q);
    return chunks ? chunks + kStepUnitCost : 0;
}

// One warp's share of chunks [c0, c1) of one head of one sequence.
template <typename T, int D, int NT>
struct StepWarp {
    static constexpr int kHalves = D / 64, kTiles = D / 16;
    static constexpr uint32_t kSideBytes = kGranule * D, kGranuleBytes = 2 * kSideBytes;
    // Of rows 8 nt + 2 t, + 1: l = sum of 2^(s - m), and o 2^e = sum of 2^(s - m) v, a weight in it being
    // 2^(s - m + power - e). m and e are whole numbers, rounded up, so that exponents add without error.
    float o[NT][kTiles][4];                // (dim pair, row)
    float m[NT][2], e[NT][2], l[NT][2];

    // `ring`: the warp's kAhead granules of shared memory; `pages`: what it knows of 64 chunks' pages.
    __device__ __forceinline__ void run(const StepArgs& p, const Sequence& q, int s, int head, int slice, int c0,
                                        int c1, uint32_t ring, StepPage* pages) {
        const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
        const Cache& c = p.a.c;
        const int rows = q.rows * p.a.group, first_seen = q.length - q.rows + 1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = e[nt][0] = e[nt][1] = kLowest, l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int mt = 0; mt < kTiles; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][mt][i] = 0.0f;
        }

        const int token_a = 4 * (g >> 1) + (g & 1);                            // of score row g; row g + 8: + 2
        const char* keys = reinterpret_cast<const char*>(c.codes) + head * c.head_pitch;
        const int stride = p.ts * kGranule, skip = slice * kGranule;
        // What the lane copies: a chunk of each of kLines tokens, kAcross lanes a token; what it reads: keys of
        // tokens token_a and token_a + 2, D / 8 values of tokens 4 t to 4 t + 3. Each is one place and, for the
        // others, a constant away or in the line's other half (xor 64).
        constexpr int kAcross = D / 16, kLines = kGranule * kAcross / 32;
        const int first = lane / kAcross * kLines;
        const char* const from = keys + first * c.token_pitch + lane % kAcross * 16;
        const uint32_t k_put = in_granule<D, false>(first, lane % kAcross), v_put = in_granule<D, true>(first, lane % kAcross);
        const uint32_t k_read = in_granule<D, false>(token_a, t);
        const uint32_t v_read = kSideBytes + in_granule<D, true>(4 * t, D == 128 ? g : g / 2) + (D == 128 ? 0 : g % 2 * 8);

        // Copies of the chunk `ahead` go to ring place `to`. Pages are looked up for 32 chunks at a time, a lane each.
        int ahead = c0;
        uint32_t to = ring;
        const auto copy = [&] {
            if (ahead < c1) {
                const int j = ahead - c0;
                if (j % 32 == 0) {
                    const int token = (ahead + lane) * stride + skip;
                    int64_t place = -1;
                    const uint32_t entry = uint32_t(__cvta_generic_to_shared(pages + j % 64 + lane));
                    __syncwarp();
                    if (ahead + lane < c1 && token < q.length) {
                        const int64_t block = ints(p.a.b.table)[s * p.a.b.table_pitch + token / c.block_size];
                        if (block < 0 || block >= c.blocks) {
                            atomicOr(p.a.status, KVSNAP_DP_BAD_BLOCK);
                        } else {
                            place = block * c.block_pitch + token % c.block_size * c.token_pitch;
                            // Its scales come with the codes: nothing waits for them here.
                            const float* scales = reinterpret_cast<const float*>(c.scales) + block * 2 * c.kv_heads + head;
                            copy_async4(entry + 8, scales);
                            copy_async4(entry + 12, scales + c.kv_heads);
                        }
                    }
                    pages[j % 64 + lane].off = place;
                    if (place < 0) pages[j % 64 + lane].ks = pages[j % 64 + lane].vs = 0.0f;
                    __syncwarp();
                }
                const int64_t found = pages[j % 64].off, at = max(found, int64_t(0));
                const bool there = found >= 0;
                __syncwarp();                            // the place's last readers are done
                const char* line = from + at;
#pragma unroll
                for (int i = 0; i < kLines; ++i) {
                    // (keys and values swizzle by other bits of the token)
                    const uint32_t k_to = D == 128 ? (to + k_put ^ i % 2 * 64) + i * 128 : to + k_put + i * 64;
                    const uint32_t v_to = D == 128 ? to + v_put + i * 128 : to + v_put ^ i * 64;
                    copy_async(k_to, line, there);
                    copy_async(v_to + kSideBytes, line + c.side_pitch, there);
                    line += c.token_pitch;
                }
                ++ahead;
                to = to == ring + (kAhead - 1) * kGranuleBytes ? ring : to + kGranuleBytes;
            }
            copies_group();
        };

#pragma unroll 1
        for (int i = 0; i < kAhead - 1; ++i) copy();

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

        uint32_t at = ring;
#pragma unroll 1
        for (int chunk = c0; chunk < c1; ++chunk) {
            copy();
            copies_done<kAhead - 1>();
            __syncwarp();
            const StepPage page = pages[(chunk - c0) % 64];
            const int base = chunk * stride + skip;

            // Two chains of products, so that one does not wait for the other.
            float sc[NT][4], odd[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[nt][i] = odd[nt][i] = 0.0f;
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
                const uint32_t read = at + k_read ^ half * 64;
                const uint4 ka = read_shared(read), kb = read_shared(read + D * 2);
                const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t a0, a1, a2, a3;
                    halves_of_codes(wa[w], a0, a2);
                    halves_of_codes(wb[w], a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma16816(w % 2 ? odd[nt] : sc[nt], a0, a1, a2, a3, qb[nt][half * 4 + w][0], qb[nt][half * 4 + w][1]);
                }
            }
            uint4 vr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (D == 128) {
                    vr[i] = read_shared(at + v_read + i * 128);
                } else {
                    const uint2 x = read_shared8((at + v_read ^ i % 2 * 64) + i / 2 * 128);
                    vr[i] = make_uint4(x.x, x.y, 0, 0);
                }
            }
            at = at == ring + (kAhead - 1) * kGranuleBytes ? ring : at + kGranuleBytes;

            // Edge: tokens that some row does not see, or a page that is not there.
            const bool dead = page.off < 0, edge = dead || base + kGranule > first_seen;
            const ValueScale vs(page.vs);
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float f = factor[nt][i] * page.ks;
                    // rounded here: fused with the subtraction of m, a score of 2^26 could exceed its own maximum by 2^4
                    sc[nt][i] = __fmul_rn(sc[nt][i] + odd[nt][i], f);
                    sc[nt][2 + i] = __fmul_rn(sc[nt][2 + i] + odd[nt][2 + i], f);
                }
            if (edge) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (dead || base + token_a >= seen[nt][i]) sc[nt][i] = -INFINITY;
                        if (dead || base + token_a + 2 >= seen[nt][i]) sc[nt][2 + i] = -INFINITY;
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    grow |= fmaxf(sc[nt][i], sc[nt][2 + i]) + fmaxf(vs.power - e[nt][i], 0.0f) > m[nt][i] + kSlack;
            if (__any_sync(~0u, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float top = fmaxf(sc[nt][i], sc[nt][2 + i]);
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
                        const float up = fmaxf(m[nt][i], ceilf(top));
                        const float same = e[nt][i] + (m[nt][i] - up);        // leaves m + e, and so o, as it is
                        l[nt][i] *= exp2_fast(m[nt][i] - up);
                        m[nt][i] = up, e[nt][i] = fmaxf(same, ceilf(top - up) + vs.power);
                        const float keep = exp2_fast(same - e[nt][i]);
#pragma unroll
                        for (int mt = 0; mt < kTiles; ++mt) o[nt][mt][i] *= keep, o[nt][mt][2 + i] *= keep;
                    }
            }
            uint32_t pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float a = sc[nt][i] - m[nt][i], b = sc[nt][2 + i] - m[nt][i], by = vs.power - e[nt][i];
                    l[nt][i] += exp2_fast(a) + exp2_fast(b);
                    w[i] = exp2_fast(a + by) * vs.part, w[2 + i] = exp2_fast(b + by) * vs.part;
                }
                pb[nt][0] = transpose8x8(pack_half2(w[0], w[1]));
                pb[nt][1] = transpose8x8(pack_half2(w[2], w[3]));
            }

            const auto add_values = [&](const uint4 (&v)[4], const uint32_t (&b)[NT][2]) {
                const uint32_t w[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w}, {v[1].x, v[1].y, v[1].z, v[1].w},
                                          {v[2].x, v[2].y, v[2].z, v[2].w}, {v[3].x, v[3].y, v[3].z, v[3].w}};
#pragma unroll
                for (int mt = 0; mt < kTiles; ++mt) {
                    const uint32_t pick = mt % 2 ? 0x7362 : 0x5140;
                    const uint32_t x = __byte_perm(w[0][mt / 2], w[1][mt / 2], pick);
                    const uint32_t y = __byte_perm(w[2][mt / 2], w[3][mt / 2], pick);
                    uint32_t a0, a1, a2, a3;
                    halves_of_codes(x, a0, a1);
                    halves_of_codes(y, a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][mt], a0, a1, a2, a3, b[nt][0], b[nt][1]);
                }
            };
            if (!edge) {
                add_values(vr, pb);
            } else if (!dead) {
                // One new token at a time, with the values it does not see left out: a weight of 0
                // times what a masked slot holds (NaN, say) must not reach it.
#pragma unroll 1
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
        }
        copies_done<0>();
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
    union {
        float o[kWarps][8 * NT][kPitch];   // once the granules are done with
        char ring[kWarps][kAhead * 2 * kGranule * D];
    };
    float2 ml[kWarps][8 * NT];
    float2 joined[8][8 * NT];              // a head's row: maximum over the slices, sum
    StepPage pages[kWarps][64];
    uint32_t sums[2][kWarps];
    uint32_t found_first;
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

    uint32_t pos = 0, end = 1, cut_total = 0;     // this CTA's part [pos, end) of what all units cost
    uint32_t from = 0;                            // where the unit's chunks begin in that
    int s = 0, hg = 0;
    Sequence q;
    if (SPLIT) {
        if (threadIdx.x == 0) p.parts.units[blockIdx.x].parts = 0;
        // What all units cost; that of up to 512 sequences are summed and found in one pass, one's need no sum.
        uint32_t mine = 0;
        if (seqs == 1) mine = cost_of(p, 0, q) * p.hg;
        else for (int i = threadIdx.x; i < seqs; i += blockDim.x) mine += cost_of(p, i, q) * p.hg;
        uint32_t sum = mine, low = 0;
        if (seqs == 1) {
            cut_total = mine;
        } else {
#pragma unroll
            for (int k = 1; k < 32; k <<= 1) {
                const uint32_t up = __shfl_up_sync(~0u, sum, k);
                if (lane >= k) sum += up;
            }
            if (lane == 31) sh.sums[0][warp] = sum;
            __syncthreads();
            for (int w = 0; w < kWarps; ++w) {
                if (w == warp) low = cut_total;
                cut_total += sh.sums[0][w];
            }
        }
        const Cut cut(cut_total, gridDim.x);
        if (blockIdx.x >= cut.ctas) return;
        pos = cut.begin(blockIdx.x), end = cut.begin(blockIdx.x + 1);
        if (seqs == 1) {
            if (threadIdx.x == 0) sh.found = 0, sh.found_first = 0;
            __syncthreads();
        } else if (seqs <= int(blockDim.x)) {
            const uint32_t first = low + sum - mine;
            if (mine && first <= pos && pos < first + mine) sh.found = threadIdx.x, sh.found_first = first;
            __syncthreads();
        } else {
            uint32_t before = 0;
            for (int tile = 0; tile < seqs && before <= pos; tile += blockDim.x) {
                const int i = tile + threadIdx.x;
                const uint32_t n = i < seqs ? cost_of(p, i, q) * p.hg : 0;
                sum = n;
#pragma unroll
                for (int k = 1; k < 32; k <<= 1) {
                    const uint32_t up = __shfl_up_sync(~0u, sum, k);
                    if (lane >= k) sum += up;
                }
                if (lane == 31) sh.sums[1][warp] = sum;
                __syncthreads();
                low = before;
                for (int w = 0; w < kWarps; ++w) {
                    if (w < warp) low += sh.sums[1][w];
                    before += sh.sums[1][w];
                }
                const uint32_t first = low + sum - n;
                if (n && first <= pos && pos < first + n) sh.found = i, sh.found_first = first;
                __syncthreads();
            }
        }
        s = sh.found;
        const uint32_t n = cost_of(p, s, q);
        hg = (pos - sh.found_first) / n;
        from = sh.found_first + hg * n + kStepUnitCost;
    } else {
        s = blockIdx.x / p.hg, hg = blockIdx.x % p.hg;
    }

    while (pos < end && s < seqs) {
        const int chunks = chunks_of(p, s, q);
        if (!chunks) {
            if (!SPLIT) return;
            ++s;
            continue;
        }
        const int c0 = SPLIT ? max(int(pos - from), 0) : 0, c1 = SPLIT ? min(chunks, int(end - from)) : chunks;
        if (c1 <= c0) return;                         // its chunks begin with the next CTA
        const int rows = q.rows * p.a.group;
        const int hc = warp % p.hc, slice = warp / p.hc;       // a warp without a slice only waits
        StepWarp<T, D, NT> w;
        if (slice < p.ts) {
            w.run(p, q, s, hg * p.hc + hc, slice, c0, c1, uint32_t(__cvta_generic_to_shared(sh.ring[warp])),
                  sh.pages[warp]);
        }
        __syncthreads();
        if (slice < p.ts) {
            const int g = lane / 4, t = lane % 4;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int n = nt * 8 + 2 * t + i;
                    if (g == 0) sh.ml[warp][n] = make_float2(w.m[nt][i], w.l[nt][i]);
                    const float by = exp2_fast(w.e[nt][i]);
#pragma unroll
                    for (int mt = 0; mt < D / 16; mt += 2)
                        *reinterpret_cast<float4*>(&sh.o[warp][n][(D / 8) * g + 2 * mt]) =
                            make_float4(w.o[nt][mt][i] * by, w.o[nt][mt][2 + i] * by, w.o[nt][mt + 1][i] * by,
                                        w.o[nt][mt + 1][2 + i] * by);
                }
            }
        }
        __syncthreads();
        // Join the slices: their factors, then 4 dims of one row and head a thread.
        for (int i = threadIdx.x; i < p.hc * rows; i += blockDim.x) {
            const int row = i % rows, h = i / rows;
            float top = kLowest, sum = 0.0f;
            for (int k = 0; k < p.ts; ++k) top = fmaxf(top, sh.ml[k * p.hc + h][row].x);
            for (int k = 0; k < p.ts; ++k) {
                float2& ml = sh.ml[k * p.hc + h][row];
                ml.x = exp2_fast(ml.x - top);
                sum += ml.x * ml.y;
            }
            sh.joined[h][row] = make_float2(top, sum);
        }
        __syncthreads();
        const bool whole = !SPLIT || (c0 == 0 && c1 == chunks);
        const int slot = 2 * int(blockIdx.x) + (c0 == 0);
        for (int i = threadIdx.x; i < p.hc * rows * (D / 4); i += blockDim.x) {
            const int at = i % (D / 4) * 4, row = i / (D / 4) % rows, h = i / (D / 4) / rows;
            float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
            for (int k = 0; k < p.ts; ++k) {
                const float f = sh.ml[k * p.hc + h][row].x;
                const float4 v = *reinterpret_cast<const float4*>(&sh.o[k * p.hc + h][row][at]);
                o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
            }
            const float2 all = sh.joined[h][row];
            const int head = hg * p.hc + h;
            if (whole) {
                // the sum is 0 only for a row that sees nothing
                const float by = all.y == 0.0f ? 0.0f : 1.0f / all.y;
                const int64_t to = int64_t(q.row + row / p.a.group) * p.a.q_heads + head * p.a.group + row % p.a.group;
                store4<T>(p.a.out + (to * D + at) * 2, make_float4(o.x * by, o.y * by, o.z * by, o.w * by));
            } else {
                const int64_t to = (int64_t(slot) * p.hc + h) * kStepRows + row;
                *reinterpret_cast<float4*>(p.parts.sums + to * D + at) = o;
                if (at == 0) p.parts.ml[to] = all;
            }
        }
        if (SPLIT) {
            if (!whole && c0 == 0 && threadIdx.x == 0) {
                const int last = Cut(cut_total, gridDim.x).of(from + chunks - 1);      // who ends the unit
                p.parts.units[blockIdx.x] = SharedUnit{q.row, hg * p.hc, 0, rows, last - int(blockIdx.x) + 1};
            }
            __syncthreads();
        }
        pos = from + c1, from = pos + kStepUnitCost;
        if (++hg == p.hg) hg = 0, ++s;
    }
}

// Joins the parts of the shared unit that a CTA of the kernels before began, which lie in consecutive CTAs'
// slots: the first CTAs those of the kernel for few rows, `first_high` of each, the others the chunks'. Where
// units have few parts (WIDE false) a warp takes a row, else a CTA does, its warps a share of the parts
// each. Bound by the way to a part and back, 4 parts at once: with nothing in the caches 5 to 6 us after steps, 14
// after 3 chunks and 18 after an 8k prompt (5000 CTAs of which most find no part), of which the launch is
// hidden behind the kernel before.
constexpr int kJoinWarps = 8;

template <typename T, int D, bool WIDE>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ AttendArgs a,
                                                               const __grid_constant__ Parts first, unsigned first_ctas,
                                                               unsigned first_high, const __grid_constant__ Parts second,
                                                               unsigned second_high) {
    constexpr int kEach = D / 32;
    using Piece = std::conditional_t<kEach == 4, float4, float2>;
    __shared__ float sums[kJoinWarps][D];
    __shared__ float stat[kJoinWarps];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const bool of_first = blockIdx.x < first_ctas * first_high;
    const Parts& p = of_first ? first : second;
    const unsigned high = of_first ? first_high : second_high, place = blockIdx.x - (of_first ? 0 : first_ctas * first_high);
    const int cta = place / high, in_high = place % high;
    const int task = WIDE ? in_high : in_high * kJoinWarps + warp;             // a row of one of the heads
    const int h = task / p.used_rows, row = task % p.used_rows;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const SharedUnit u = p.units[cta];
    if (u.parts == 0 || h >= p.heads || row >= u.rows) return;
    const int slot_rows = p.heads * p.head_rows, in = h * p.head_rows + row;
    const auto at = [&](int f) { return int64_t(2 * (cta + f) + (f == 0)) * slot_rows + in; };
    const auto part = [&](int f) { return *reinterpret_cast<const Piece*>(p.sums + at(f) * D + lane * kEach); };
    float o[kEach] = {}, top = kLowest, sum = 0.0f;
    const auto add = [&](const Piece& v, float by) {
        const float* x = reinterpret_cast<const float*>(&v);
#pragma unroll
        for (int i = 0; i < kEach; ++i) o[i] += by * x[i];
    };
    // The maximum of all parts; then a warp's parts (of WIDE every eighth), 4 on their way at a time.
    for (int i = lane; i < u.parts; i += 32) top = fmaxf(top, p.ml[at(i)].x);
    const int begin = WIDE ? warp : 0, step = WIDE ? kJoinWarps : 1;
    for (int i = begin; i < u.parts; i += 4 * step) {
        Piece v[4];
        float2 ml[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int f = min(i + j * step, u.parts - 1);
            v[j] = part(f), ml[j] = p.ml[at(f)];
        }
        if (i == begin) top = warp_max(top);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float by = i + j * step < u.parts ? exp2_fast(ml[j].x - top) : 0.0f;
            add(v[j], by);
            sum += by * ml[j].y;
        }
    }
    if (WIDE) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) sums[warp][lane * kEach + i] = o[i];
        if (lane == 0) stat[warp] = sum;
        __syncthreads();
        if (warp) return;
        sum = 0.0f;
        for (int w = 0; w < kJoinWarps; ++w) sum += stat[w];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            o[i] = 0.0f;
            for (int w = 0; w < kJoinWarps; ++w) o[i] += sums[w][lane * kEach + i];
        }
    }
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int r = u.first + row;
    const int64_t to = int64_t(u.row + r / a.group) * a.q_heads + (u.head + h) * a.group + r % a.group;
    char* out = a.out + (to * D + lane * kEach) * 2;
    if constexpr (kEach == 4) store4<T>(out, make_float4(o[0] * by, o[1] * by, o[2] * by, o[3] * by));
    else *reinterpret_cast<uint32_t*>(out) = T::pack(o[0] * by, o[1] * by);
}

// ---- many rows: chunks and prompts --------------------------------------------------------
//
// Sequences that the kernel above does not take. 4 D operations a query head and visible token, in two
// products of fp16 operands with 32-bit sums in tensor memory: 0.67 to 0.71 ms for an 8k prompt of 32 heads
// of 128, 770 to 820 TFLOP/s, half of what a plain product reaches. What bounds it are the softmax warps: the
// weights' exponentials and what surrounds them take about 1980 clocks a step of both row tiles, the
// tensor cores' part 1300. Chunks that do not fill 256 rows pay for the rows that they lack.
// A CTA takes 256 rows (two tiles of 128) of one KV head in steps of 64 tokens:
//   warp 13     looks up the pages of coming steps and their scales;
//   warps 8-11  load a step's codes, one step ahead, turn them to fp16 and lay them out for the tensor
//               cores; both row tiles use them, so a code is converted once per 256 rows;
//   warp 12     issues S = Q K^T and O += P V, the scores two steps ahead of the sums, so that a
//               row tile's next scores are there when its softmax of these ends;
//   warps 0-7   a thread a row: maximum, weights, sums; P goes back to tensor memory over S.
// Tensor memory holds exactly this: two tiles' sums (2 x 128 columns) and two steps of scores of each
// (4 x 64). With one step of 128 tokens instead, scores and softmax took turns: 1.02 ms for an 8k
// prompt of 32 heads.
// The running maximum follows a row's true maximum only when that exceeds it by 2^14 (weights stay
// within fp16), so sums in tensor memory are rarely touched (followed at every step: an 8k prompt 780 us,
// so 669). A page's scale goes into the conversion relative to the largest of its step, where e4m3's
// 9 fraction bits below 1 leave fp16 room: keys down to 2^-14, values down to 2^-6. The step's key scale
// multiplies S, its value scale the weights, relative to a running maximum of their products (a row's e:
// O 2^e are the sums). Steps whose pages lie further apart take their pages' own scales into
// the scores instead, and sum their weights apart.

constexpr int kTile = 128;                 // rows a tile
constexpr int kUnitRows = 2 * kTile;
constexpr int kStep = 64;                  // tokens a step
constexpr int kGranules = kStep / kGranule;
constexpr int kStages = 4;                 // steps of keys and of values in shared memory
// What a unit costs besides its steps (queries in, sums out, the pipeline's filling), in steps: work is
// cut by steps and this (by steps alone an 8k prompt takes 770 us, so 669, and 24 chunks of 128 tokens 270, so
// 185: a CTA with many short units was 1.6 times as long as others).
constexpr int kUnitCost = 8;
constexpr int kConvertWarps = 4, kIssueWarp = 12, kLookWarp = 13, kChunkThreads = 512;
constexpr int kLooked = 16;                // steps looked up ahead
constexpr int kScales = 8;                 // steps whose scales the softmax may still need
constexpr int kLookedUnits = 4;            // units
constexpr float kKeysApart = 1.0f / 16384;  // a step's smallest key scale to its largest, and powers of value
constexpr float kValuesApart = 6.0f;       // scales, up to which the conversion takes them
constexpr float kFarBelow = 60.0f;         // powers of two below a row's e from which weights are summed apart
constexpr float kLargeScore = 1048576.0f;  // size of scores from which they are rounded before m is taken away
constexpr uint32_t kSumsAt = 256;          // columns of tensor memory: S and P 0 to 255, O from here

struct ChunkArgs {
    AttendArgs a;
    Parts parts;
};

// One tile of a unit: its place in the work, the same for every role of the CTA.
struct Unit {
    Sequence q;
    int s, head, tile;        // sequence, KV head, tile of 256 rows
    int first, rows;          // its rows of the head
    int first_seen;           // tokens that its first row sees
    int steps;                // that its last row sees
};

__device__ __forceinline__ bool chunk_sequence(const AttendArgs& a, int s, Sequence& q) {
    return read_sequence(a.b, a.c.block_size, s, q, a.status) && q.rows * a.group > a.step_rows;
}

__device__ __forceinline__ int steps_of(const AttendArgs& a, const Sequence& q, int tile) {
    const int last = min(q.rows * a.group, (tile + 1) * kUnitRows) - 1;
    const int seen = q.length - q.rows + last / a.group + 1;
    return max(1, (seen + kStep - 1) / kStep);
}

__device__ __forceinline__ int row_tiles(const AttendArgs& a, const Sequence& q) {
    return (q.rows * a.group + kUnitRows - 1) / kUnitRows;
}

// Cost of one head of sequence s in steps, summed by a warp.
__device__ __forceinline__ int64_t head_cost(const AttendArgs& a, int s) {
    Sequence q;
    if (!chunk_sequence(a, s, q)) return 0;
    int64_t n = 0;
    for (int i = threadIdx.x % 32; i < row_tiles(a, q); i += 32) n += kUnitCost + steps_of(a, q, i);
#pragma unroll
    for (int k = 16; k; k >>= 1) n += __shfl_xor_sync(~0u, n, k);
    return n;
}

constexpr int kScanned = 256;              // sequences scanned at a time
constexpr int kNanUnits = 64;              // more units than the roles can be apart

constexpr uint32_t kAllLive = (1u << kGranules) - 1, kApart = 1u << kGranules;

// What a step's conversion needs to know.
struct Looked {
    int64_t keys[kGranules];               // addresses of the granules' key codes; 0: not there
    uint32_t k_by[kGranules], v_by[kGranules];   // what their codes are multiplied by, as fp16 pairs
    float k_scale, v_power;                // largest key scale of the step; power of its largest value scale
    uint32_t live;                         // granules that are there; kApart: their own scales count
    float k_own[kGranules], v_own[kGranules];    // with kApart: their key scales, and powers less v_power
    int tokens;                            // of the step that the sequence has
    int edge;                              // some row does not see all of them
    int last;                              // of the CTA
    int unit;
};

// What the other roles need to know of a unit, and of the steps [begin, end) of it that are this CTA's.
struct LookedUnit {
    Sequence q;
    int s, head, first, rows, first_seen, steps, begin, end;
    int last;                              // of this CTA
    int64_t stop;                          // where it ends in all the work
};

struct ChunkControl {
    uint64_t q_full[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t s_full[2][2], p_full[2][2], o_full[2][2], drained;    // of a row tile; of a step's turn
    uint64_t looked[kLooked], look_free[kLooked];
    Looked look[kLooked];
    uint64_t unit_looked[kLookedUnits], unit_free[kLookedUnits];
    LookedUnit unit[kLookedUnits];
    float k_scale[kScales], v_power[kScales];    // of a step, as in Looked
    uint32_t live[kScales];
    float k_own[kScales][kGranules], v_own[kScales][kGranules];
    int nan_unit[kNanUnits];               // a unit (counted from 1) whose last steps hold a NaN value
    uint32_t tensor;                       // tensor memory's address
    volatile int stop;                     // a wait ran out
    int64_t counts[kScanned], scratch[32];
    int64_t total, pos, until, base, sought, scanned;      // pos to until: this CTA's part of the total cost
    int s, head, tile;
};

template <int D>
struct ChunkShared {
    char q[2][kTile * D * 2];
    char k[kStages][kStep * D * 2];
    char v[kStages][kStep * D * 2];
    ChunkControl c;
};

// The look-up's way through the units that a CTA has steps of.
struct Walk {
    int64_t base, stop;       // where the unit begins in all the work, and where the CTA's work ends, in cost
    int begin, end;           // steps of the unit that are this CTA's
    int unit;                 // counted from 0
    Unit u;

    // The unit that u names, from place `from` on; false without a step in it.
    __device__ __forceinline__ bool load(const AttendArgs& a, int64_t from) {
        u.first = u.tile * kUnitRows;
        u.rows = min(u.q.rows * a.group - u.first, kUnitRows);
        u.first_seen = u.q.length - u.q.rows + u.first / a.group + 1;
        u.steps = steps_of(a, u.q, u.tile);
        begin = int(max(int64_t(0), from - base - kUnitCost));
        end = int(min(int64_t(u.steps), stop - base - kUnitCost));
        return end > begin;
    }
    __device__ __forceinline__ bool next(const AttendArgs& a) {
        do {
            base += kUnitCost + u.steps;
            if (base >= stop) return false;
            if (++u.tile >= row_tiles(a, u.q)) {
                u.tile = 0;
                if (++u.head == a.c.kv_heads) {
                    u.head = 0;
                    for (++u.s; u.s < a.b.seqs && !chunk_sequence(a, u.s, u.q); ++u.s) {}
                    if (u.s >= a.b.seqs) return false;
                }
            }
        } while (!load(a, base));
        ++unit;
        return true;
    }
    __device__ __forceinline__ bool start(const AttendArgs& a, const ChunkControl& c) {
        base = c.base, stop = c.until, unit = -1;
        u.s = c.s, u.head = c.head, u.tile = c.tile;
        if (!chunk_sequence(a, u.s, u.q)) return false;
        if (!load(a, c.pos)) return next(a);
        unit = 0;
        return true;
    }
};

__device__ __forceinline__ uint32_t shared_address(const void* p) {
    return uint32_t(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void barrier_init(uint64_t* b, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(b)), "r"(count) : "memory");
}

__device__ __forceinline__ void barrier_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(shared_address(b)) : "memory");
}

// Waits for the barrier's phase of this parity; false after about two seconds, or (unless `last`)
// once another wait ran out.
__device__ __forceinline__ bool barrier_wait(uint64_t* b, uint32_t parity, ChunkControl& c, bool last = false) {
    const uint32_t at = shared_address(b);
    uint64_t began = 0;
    for (int i = 0;; ++i) {
        uint32_t done;
        asm volatile("{\n.reg .pred p;\n"
                     "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
                     "selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(done) : "r"(at), "r"(parity) : "memory");
        if (done) return true;
        if (i % 256 == 255) {
            uint64_t now;
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
            if (!began) began = now;
            if ((c.stop && !last) || now - began > 2000000000ull) {
                c.stop = 1;
                return false;
            }
        }
    }
}

__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity, ChunkControl& c) {
    return __all_sync(~0u, barrier_wait(b, parity, c));
}

// The tensor cores' instructions are issued by one lane, `chosen`, of a warp that goes through the code
// as a whole, so that addresses stay in uniform registers: built by a lane alone, each instruction took
// 70 to 110 clocks to issue, for 32 to 64 of work.
__device__ __forceinline__ void commit(uint64_t* b, uint32_t chosen) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %1, 0;\n"
                 "@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}"
                 ::"r"(shared_address(b)), "r"(chosen) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A matrix in shared memory in rows of 128 bytes, 128-byte swizzled in groups of 8 rows (1 KiB).
// By rows of K (keys, queries): a row is 64 of the contracted elements, `lead` is not used.
// By rows of N (values): a row is 64 columns of one contracted element; `lead` is the way to the next 64.
// Low word of its description; the high one is the same for all.
__device__ __forceinline__ uint32_t matrix(uint32_t at, uint32_t lead) { return at >> 4 | lead >> 4 << 16; }
constexpr uint32_t kMatrixHigh = 1024 >> 4 | 1 << 14 | 2 << 29;

// 128 x n products of fp16 with 32-bit sums; by_n: B lies by rows of N.
__host__ __device__ constexpr uint32_t instruction(int n, bool by_n) {
    return 1u << 4 | uint32_t(by_n) << 16 | uint32_t(n >> 3) << 17 | uint32_t(kTile >> 4) << 24;
}

__device__ __forceinline__ void mma_shared(uint32_t d, uint32_t a, uint32_t b, uint32_t what, uint32_t add,
                                           uint32_t chosen) {
    asm volatile("{\n.reg .pred p, q;\n.reg .b64 a, b;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
                 "mov.b64 a, {%1, %6};\nmov.b64 b, {%2, %6};\n"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}"
                 ::"r"(d), "r"(a), "r"(b), "r"(what), "r"(add), "r"(chosen), "r"(kMatrixHigh) : "memory");
}

__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint32_t b, uint32_t what, uint32_t add,
                                           uint32_t chosen) {
    asm volatile("{\n.reg .pred p, q;\n.reg .b64 b;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
                 "mov.b64 b, {%2, %6};\n"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}"
                 ::"r"(d), "r"(a), "r"(b), "r"(what), "r"(add), "r"(chosen), "r"(kMatrixHigh) : "memory");
}

// Columns of the warp's 32 rows of tensor memory, a row a lane.
__device__ __forceinline__ void tensor_load(uint32_t at, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
          "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
          "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(at));
}

__device__ __forceinline__ void tensor_load(uint32_t at, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(at));
}

// The loads so far, and that `v` comes from them.
__device__ __forceinline__ void tensor_loaded(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
          "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
        :: "memory");
}

__device__ __forceinline__ void tensor_store(uint32_t at, const float (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        :: "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]),
          "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]),
          "r"(at) : "memory");
}

__device__ __forceinline__ void tensor_load(uint32_t at, float (&v)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,"
        "%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,"
        "%56,%57,%58,%59,%60,%61,%62,%63"
        "}, [%64];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]),
          "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]),
          "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]),
          "=f"(v[29]), "=f"(v[30]), "=f"(v[31]), "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]),
          "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]), "=f"(v[40]), "=f"(v[41]), "=f"(v[42]),
          "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]), "=f"(v[48]), "=f"(v[49]),
          "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]), "=f"(v[56]),
          "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
        : "r"(at));
}

// The loads so far, and that `v` comes from them.
__device__ __forceinline__ void tensor_loaded(float (&v)[64]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
          "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
          "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
          "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]),
          "+f"(v[29]), "+f"(v[30]), "+f"(v[31]), "+f"(v[32]), "+f"(v[33]), "+f"(v[34]), "+f"(v[35]),
          "+f"(v[36]), "+f"(v[37]), "+f"(v[38]), "+f"(v[39]), "+f"(v[40]), "+f"(v[41]), "+f"(v[42]),
          "+f"(v[43]), "+f"(v[44]), "+f"(v[45]), "+f"(v[46]), "+f"(v[47]), "+f"(v[48]), "+f"(v[49]),
          "+f"(v[50]), "+f"(v[51]), "+f"(v[52]), "+f"(v[53]), "+f"(v[54]), "+f"(v[55]), "+f"(v[56]),
          "+f"(v[57]), "+f"(v[58]), "+f"(v[59]), "+f"(v[60]), "+f"(v[61]), "+f"(v[62]), "+f"(v[63])
        :: "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Two products and sums, or sums, in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 a, b, c;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
        "fma.rn.f32x2 a, a, b, c;\nmov.b64 {%0, %1}, a;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 a, b;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\n"
        "add.rn.f32x2 a, a, b;\nmov.b64 {%0, %1}, a;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ void tensor_loaded(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
          "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
          "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]),
          "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
        :: "memory");
}

__device__ __forceinline__ void tensor_store(uint32_t at, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        :: "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
          "r"(at) : "memory");
}

__device__ __forceinline__ void tensor_store(uint32_t at, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
        :: "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(at) : "memory");
}

__device__ __forceinline__ void tensor_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Where 16 bytes (8 fp16) `chunk` of row r lie in a matrix of R rows of fp16.
template <int R>
__device__ __forceinline__ uint32_t swizzled(int r, int chunk) {
    return uint32_t(chunk / 8) * (R * 128) + uint32_t(r) * 128 + uint32_t((chunk % 8) ^ (r % 8)) * 16;
}

__device__ __forceinline__ void store_shared(char* at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    *reinterpret_cast<uint4*>(at) = make_uint4(a, b, c, d);
}

__device__ __forceinline__ uint32_t times_half2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// The role of warp 13: 8 steps at a time, a lane a granule.
__device__ __forceinline__ void look_role(const ChunkArgs& p, ChunkControl& c, Walk w) {
    constexpr int kParts = 32 / kGranules;
    const AttendArgs& a = p.a;
    const Cache& cache = a.c;
    const int lane = threadIdx.x % 32, part = lane / kGranules, granule = lane % kGranules;
    for (int64_t it = 0;;) {
        Walk after = w;
        const bool more = after.next(a);
        const int k = w.unit % kLookedUnits;
        if (!warp_wait(&c.unit_free[k], uint32_t(w.unit / kLookedUnits + 1) % 2, c)) return;
        if (lane == 0) {
            c.unit[k] = LookedUnit{w.u.q, w.u.s, w.u.head, w.u.first, w.u.rows, w.u.first_seen, w.u.steps, w.begin,
                                   w.end, !more, w.base + kUnitCost + w.u.steps};
            barrier_arrive(&c.unit_looked[k]);
        }
        // Its queries come to the L2 meanwhile.
        for (int i = lane; i < w.u.rows; i += 32) {
            const int r = w.u.first + i;
            const char* at = a.query.at + int64_t(w.u.q.row + r / a.group) * a.query.token +
                             int64_t(w.u.head * a.group + r % a.group) * a.query.head;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
            if (cache.head_dim > 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + 128));
        }
        for (int first = w.begin; first < w.end; first += kParts) {
            const int n = min(kParts, w.end - first), step = first + part;
            const int64_t token = int64_t(step) * kStep + granule * kGranule;
            int64_t at = 0;
            float ks = 0.0f, vs = 0.0f;
            if (part < n && token < w.u.q.length) {
                const int64_t block = ints(a.b.table)[w.u.s * a.b.table_pitch + token / cache.block_size];
                if (block < 0 || block >= cache.blocks) {
                    atomicOr(a.status, KVSNAP_DP_BAD_BLOCK);
                } else {
                    at = cache.codes + block * cache.block_pitch + token % cache.block_size * cache.token_pitch +
                         w.u.head * cache.head_pitch;
                    const float* scales = reinterpret_cast<const float*>(cache.scales) + block * 2 * cache.kv_heads + w.u.head;
                    ks = scales[0], vs = scales[cache.kv_heads];
                }
            }
            const ValueScale v(vs);
            float k_top = ks, v_top = v.power;
#pragma unroll
            for (int i = kGranules / 2; i; i >>= 1) {
                k_top = fmaxf(k_top, __shfl_xor_sync(~0u, k_top, i));
                v_top = fmaxf(v_top, __shfl_xor_sync(~0u, v_top, i));
            }
            v_top = fmaxf(v_top, -126.0f);             // of no values but zeros: any finite one
            const bool far = at && ((ks > 0.0f && ks < k_top * kKeysApart) || v.power < v_top - kValuesApart);
            const uint32_t live = __ballot_sync(~0u, at != 0) >> (kGranules * part) & kAllLive;
            const bool apart = __ballot_sync(~0u, far) >> (kGranules * part) & kAllLive;
            const __half2 k_by = __float2half2_rn(apart ? 1.0f : k_top > 0.0f ? ks / k_top : 0.0f);
            const __half2 v_by = __float2half2_rn(apart ? v.part : v.part * exp2_fast(v.power - v_top));
            for (int i = 0; i < n; ++i)
                if (!warp_wait(&c.look_free[(it + i) % kLooked], uint32_t((it + i) / kLooked + 1) % 2, c)) return;
            if (part < n) {
                Looked& to = c.look[(it + part) % kLooked];
                to.keys[granule] = at;
                to.k_by[granule] = reinterpret_cast<const uint32_t&>(k_by);
                to.v_by[granule] = reinterpret_cast<const uint32_t&>(v_by);
                to.k_own[granule] = ks, to.v_own[granule] = v.power - v_top;
                if (granule == 0) {
                    to.k_scale = k_top, to.v_power = v_top, to.live = live | (apart ? kApart : 0);
                    to.tokens = int(min(int64_t(kStep), max(int64_t(0), w.u.q.length - token)));
                    to.edge = int64_t(step + 1) * kStep > w.u.first_seen;
                    to.last = !more && step + 1 == w.end;
                    to.unit = w.unit;
                }
            }
            __syncwarp();
            if (lane < n) barrier_arrive(&c.looked[(it + lane) % kLooked]);
            it += n;
        }
        if (!more) return;
        w = after;
    }
}

// The role of warps 8-11.
template <int D>
__device__ __forceinline__ void convert_role(const ChunkArgs& p, ChunkShared<D>& sh) {
    constexpr int kAcross = D / 16, kTokens = 32 * kConvertWarps / kAcross, kEach = kStep / kTokens;
    const Cache& c = p.a.c;
    const int tid = threadIdx.x - 256, lane = threadIdx.x % 32;
    // A thread's 16 codes: token my_token + i * kTokens, dims 16 * piece. Of 8 consecutive lanes
    // 4 are an even and 4 an odd token, so their swizzled 16-byte stores meet all banks.
    const int my_token = D == 128 ? tid / 16 * 2 + tid / 4 % 2 : tid / 4;
    const int piece = D == 128 ? tid % 4 + tid / 8 % 2 * 4 : tid % 4;
    const int64_t within = my_token % kGranule * c.token_pitch + 16 * piece;

    // Keys and values in turn, the next load on its way while one is converted.
    const auto load = [&](uint4 (&to)[kEach], int64_t step, int64_t side) {
        const Looked& look = sh.c.look[step % kLooked];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int token = my_token + i * kTokens;
            const int64_t at = look.keys[token / kGranule];
            // Slots behind the last token hold anything, NaN included: they count as zeros.
            to[i] = load16(reinterpret_cast<const char*>(at) + side + within, at && token < look.tokens);
        }
    };
    const auto convert = [&](const uint4 (&from)[kEach], char* to, const uint32_t* by) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int token = my_token + i * kTokens;
            const uint32_t f = by[token / kGranule];
            const uint32_t x[4] = {from[i].x, from[i].y, from[i].z, from[i].w};
            uint32_t h[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                halves_of_codes(x[j], h[2 * j], h[2 * j + 1]);
                h[2 * j] = times_half2(h[2 * j], f), h[2 * j + 1] = times_half2(h[2 * j + 1], f);
            }
            store_shared(to + swizzled<kStep>(token, 2 * piece), h[0], h[1], h[2], h[3]);
            store_shared(to + swizzled<kStep>(token, 2 * piece + 1), h[4], h[5], h[6], h[7]);
        }
        fence_shared();
        __syncwarp();
    };
    // One step, with the next one's loads on their way: true where there is a next one.
    const auto turn = [&](uint4 (&kr)[kEach], uint4 (&vr)[kEach], uint4 (&k_next)[kEach], uint4 (&v_next)[kEach],
                          int64_t step) {
        const int slot = step % kStages;
        const uint32_t free = uint32_t(step / kStages + 1) % 2;
        const Looked& look = sh.c.look[step % kLooked];
        const bool more = !look.last;
        if (tid == 0) {
            sh.c.k_scale[step % kScales] = look.k_scale, sh.c.v_power[step % kScales] = look.v_power;
            sh.c.live[step % kScales] = look.live;
            if (look.live & kApart)
                for (int i = 0; i < kGranules; ++i)
                    sh.c.k_own[step % kScales][i] = look.k_own[i], sh.c.v_own[step % kScales][i] = look.v_own[i];
        }
        if (!warp_wait(&sh.c.k_empty[slot], free, sh.c)) return false;
        convert(kr, sh.k[slot], look.k_by);
        if (lane == 0) barrier_arrive(&sh.c.k_full[slot]);
        if (more) {
            if (!warp_wait(&sh.c.looked[(step + 1) % kLooked], uint32_t((step + 1) / kLooked) % 2, sh.c)) return false;
            load(k_next, step + 1, 0);
            load(v_next, step + 1, c.side_pitch);
        }
        if (look.edge) {
            // Some row does not see some of these tokens, and a weight of 0 times NaN is NaN: NaN
            // values are left out here, and put back at the end into the rows that see them.
            bool found = false;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                uint32_t x[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t bad = ((x[j] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                    found |= bad != 0;
                    x[j] &= ~((bad >> 7) * 0xFFu);
                }
                vr[i] = make_uint4(x[0], x[1], x[2], x[3]);
            }
            if (found) sh.c.nan_unit[look.unit % kNanUnits] = look.unit + 1;
        }
        if (!warp_wait(&sh.c.v_empty[slot], free, sh.c)) return false;
        convert(vr, sh.v[slot], look.v_by);
        if (lane == 0) {
            barrier_arrive(&sh.c.v_full[slot]);
            barrier_arrive(&sh.c.look_free[step % kLooked]);
        }
        return more;
    };
    // Two steps' registers by turns: copies between them would wait for the loads.
    uint4 ka[kEach], va[kEach], kb[kEach], vb[kEach];
    if (!warp_wait(&sh.c.looked[0], 0, sh.c)) return;
    load(ka, 0, 0);
    load(va, 0, c.side_pitch);
#pragma unroll 1
    for (int64_t step = 0;; step += 2)
        if (!turn(ka, va, kb, vb, step) || !turn(kb, vb, ka, va, step + 1)) return;
}

// The role of warp 12.
template <int D>
__device__ __forceinline__ void issue_role(ChunkShared<D>& sh) {
    constexpr uint32_t kScores = instruction(kStep, false), kSums = instruction(D, true);
    const uint32_t tensor = __shfl_sync(~0u, sh.c.tensor, 0);
    uint32_t chosen;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(chosen));
    const uint32_t q_at = matrix(shared_address(sh.q[0]), 16), k_at = matrix(shared_address(sh.k[0]), 16);
    const uint32_t v_at = matrix(shared_address(sh.v[0]), kStep * 128);
    // S of a row tile's step, in the half of its columns that the step's turn gives.
    const auto scores = [&](uint32_t tile, uint32_t step, uint32_t turn) {
        const uint32_t d = tensor + tile * kTile + turn % 2 * kStep;
        const uint32_t q = q_at + tile * (sizeof(sh.q[0]) >> 4), k = k_at + step % kStages * (sizeof(sh.k[0]) >> 4);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
            mma_shared(d, q + ((i / 4 * kTile * 128 + i % 4 * 32) >> 4), k + ((i / 4 * kStep * 128 + i % 4 * 32) >> 4),
                       kScores, i > 0, chosen);
        commit(&sh.c.s_full[tile][turn % 2], chosen);
    };
    const auto sums = [&](uint32_t tile, uint32_t step, uint32_t turn, bool add) {
        const uint32_t d = tensor + kSumsAt + tile * kTile, p = tensor + tile * kTile + turn % 2 * kStep;
        const uint32_t v = v_at + step % kStages * (sizeof(sh.v[0]) >> 4);
#pragma unroll
        for (int i = 0; i < kStep / 16; ++i)
            mma_tensor(d, p + 8 * i, v + (i * 2048 >> 4), kSums, add || i > 0, chosen);
        commit(&sh.c.o_full[tile][turn % 2], chosen);
    };
    uint32_t it = 0;
    uint32_t turn0 = 0, turn1 = 0, q_turn0 = 0, q_turn1 = 0;     // steps and units that each row tile has had
    for (uint32_t unit = 0;; ++unit) {
        if (!warp_wait(&sh.c.unit_looked[unit % kLookedUnits], unit / kLookedUnits % 2, sh.c)) return;
        const LookedUnit& u = sh.c.unit[unit % kLookedUnits];
        const bool both = __shfl_sync(~0u, u.rows, 0) > kTile, final = __shfl_sync(~0u, u.last, 0);
        const int n = __shfl_sync(~0u, u.end - u.begin, 0);
        if (chosen) barrier_arrive(&sh.c.unit_free[unit % kLookedUnits]);
        if (!warp_wait(&sh.c.q_full[0], q_turn0++ % 2, sh.c)) return;
        if (both && !warp_wait(&sh.c.q_full[1], q_turn1++ % 2, sh.c)) return;
        // A step's sums, then the scores of the step after the next, which take the columns of its weights.
#pragma unroll 1
        for (int step = -2; step < n; ++step) {
            const uint32_t now = it + step, ahead = it + step + 2;
            const bool more = step + 2 < n;
            if (step >= 0) {
                if (!warp_wait(&sh.c.p_full[0][turn0 % 2], turn0 / 2 % 2, sh.c)) return;
                if (!warp_wait(&sh.c.v_full[now % kStages], now / kStages % 2, sh.c)) return;
                fence_after();
                sums(0, now, turn0, step > 0);
                if (!both) commit(&sh.c.v_empty[now % kStages], chosen);
            }
            if (more) {
                if (!warp_wait(&sh.c.k_full[ahead % kStages], ahead / kStages % 2, sh.c)) return;
                fence_after();
                scores(0, ahead, step >= 0 ? turn0 + 2 : turn0 + step + 2);
                if (!both) commit(&sh.c.k_empty[ahead % kStages], chosen);
            }
            if (both) {
                if (step >= 0) {
                    if (!warp_wait(&sh.c.p_full[1][turn1 % 2], turn1 / 2 % 2, sh.c)) return;
                    fence_after();
                    sums(1, now, turn1, step > 0);
                    commit(&sh.c.v_empty[now % kStages], chosen);
                }
                if (more) {
                    scores(1, ahead, step >= 0 ? turn1 + 2 : turn1 + step + 2);
                    commit(&sh.c.k_empty[ahead % kStages], chosen);
                }
            }
            if (step >= 0) ++turn0, turn1 += both;
        }
        it += n;
        if (final) return;
    }
}

// 16 bytes `chunk` of a row in a warp's 4 KB of shared memory: 32 rows of 128 bytes, in which rows that
// came a lane a row go out 8 lanes a row.
__device__ __forceinline__ char* staged(char* warp_rows, int row, int chunk) {
    return warp_rows + row * 128 + (chunk ^ row % 8) * 16;
}

// What a softmax thread knows of its row: l = sum of 2^(s - m); sums in tensor memory, times 2^e, = sum of
// 2^(s - m) v. Whole numbers m and e, as in StepWarp.
struct RowState {
    float m, e, l;
};

constexpr float kLeast = 1.17549435e-38f;  // the smallest normal number

__device__ __forceinline__ bool large_score(float s) { return fabsf(s) > kLargeScore && s > kLowest / 2; }

// Multiplies the sums so far in tensor memory, once the step before is in them.
template <int D>
__device__ __forceinline__ bool rescale(uint32_t sums, float keep, uint64_t* summed, uint32_t parity, ChunkControl& c) {
    if (!warp_wait(summed, parity, c)) return false;
    fence_after();
#pragma unroll 1
    for (int i = 0; i < D / 16; ++i) {
        float y[16];
        __syncwarp();                                    // lanes meet before each access to tensor memory
        tensor_load(sums + 16 * i, y);
        tensor_loaded(y);
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] *= keep;
        tensor_store(sums + 16 * i, y);
    }
    return true;
}

// A step whose weights in the sums do not tell those of l: a granule of 16 columns at a time, three times, from
// scores that are rounded before m is taken away. `k_own`: pages by their own scales. Weights take columns that
// have been read. Out of line, as the loop over steps is to stay in the instruction cache: an 8k prompt takes
// 697 us, with this in the loop's way 731, without it at all 689.
template <int D>
__device__ __noinline__ bool step_alone(RowState& row, uint32_t at, uint64_t seen, const float* k_own, const float* v_own,
                                        float factor, float f, float power, uint32_t sums, uint64_t* summed,
                                        uint32_t parity, ChunkControl& c) {
    float m = row.m, e = row.e, top = -INFINITY, sum = 0.0f, by = 0.0f;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
#pragma unroll 1
        for (int i = 0; i < kGranules; ++i) {
            float y[kGranule];
            __syncwarp();
            tensor_load(at + kGranule * i, y);
            const float k = k_own ? fmaxf(factor * k_own[i], kLeast) : f, v = k_own ? v_own[i] : 0.0f;
            const uint32_t see = uint32_t(seen >> (kGranule * i));
            tensor_loaded(y);
#pragma unroll
            for (int j = 0; j < kGranule; ++j) y[j] = see >> j & 1 ? __fmul_rn(y[j], k) : -INFINITY;
            if (pass == 0) {
#pragma unroll
                for (int j = 0; j < kGranule; ++j) top = fmaxf(top, y[j]);
            } else if (pass == 1) {
#pragma unroll
                for (int j = 0; j < kGranule; ++j) {
                    y[j] -= m;
                    sum += exp2_fast(y[j]), top = fmaxf(top, y[j] + v);
                }
            } else {
                uint32_t weights[kGranule / 2];
#pragma unroll
                for (int j = 0; j < kGranule; ++j) y[j] = exp2_fast(y[j] - m + (v + by));
#pragma unroll
                for (int j = 0; j < kGranule / 2; ++j) weights[j] = pack_half2(y[2 * j], y[2 * j + 1]);
                __syncwarp();
                tensor_store(at + kGranule / 2 * i, weights);
            }
        }
        if (pass == 0) {
            if (top > m) {                               // leaves m + e, and so the sums, as they are
                const float up = ceilf(top);
                row.l *= exp2_fast(m - up);
                e += m - up, m = up;
            }
            top = -INFINITY;
        } else if (pass == 1) {
            float keep = 1.0f;
            if (top + power > e + kSlack) {
                const float up = ceilf(top) + power;
                keep = exp2_fast(e - up);
                e = up;
            }
            if (summed && __any_sync(~0u, keep != 1.0f) && !rescale<D>(sums, keep, summed, parity, c)) return false;
            by = power - e;
        }
    }
    row.m = m, row.e = e, row.l += sum;
    return true;
}

// The role of warps 0-3 (row tile 0) and 4-7 (row tile 1).
template <typename T, int D>
__device__ __forceinline__ void softmax_role(const ChunkArgs& p, ChunkShared<D>& sh) {
    constexpr int kLanes = D / 8;                        // lanes of 8 elements that a row takes
    const AttendArgs& a = p.a;
    const int tile = threadIdx.x / 128, r = threadIdx.x % 128, lane = threadIdx.x % 32, warp_row = r - lane;
    const uint32_t scores = sh.c.tensor + (uint32_t(warp_row) << 16) + tile * kTile, sums = scores + kSumsAt;
    uint32_t it = 0, turn = 0;
    for (uint32_t unit = 0;; ++unit) {
        const int ring = unit % kLookedUnits;
        if (!warp_wait(&sh.c.unit_looked[ring], unit / kLookedUnits % 2, sh.c)) return;
        const LookedUnit& u = sh.c.unit[ring];
        const bool final = u.last;
        const int begin = u.begin, end = u.end;
        if (tile * kTile >= u.rows) {                    // no rows for this tile: its steps pass by
            it += end - begin;
            __syncwarp();
            if (lane == 0) barrier_arrive(&sh.c.unit_free[ring]);
            if (final) return;
            continue;
        }
        const int rows = min(u.rows - tile * kTile - warp_row, 32);        // of this warp (may be none)
        const int row = u.first + tile * kTile + r, token = row / a.group;
        const int seen = lane < rows ? u.q.length - u.q.rows + token + 1 : 0;

        // The queries as fp16, a row times a power of two that brings its largest element to [2^14, 2^15).
        // They come in D / 8 lanes a row, so that whole lines are read; then a lane takes a row.
        const int out_row = (u.q.row + token) * a.q_heads + u.head * a.group + row % a.group;
        float factor;
        {
            const int64_t mine = int64_t(u.q.row + token) * a.query.token +
                                 int64_t(u.head * a.group + row % a.group) * a.query.head;
            char* const to = sh.q[tile];
            uint4 raw[kLanes];
#pragma unroll
            for (int i = 0; i < kLanes; ++i) {
                const int x = i * (32 / kLanes) + lane / kLanes;
                const int64_t at = __shfl_sync(~0u, mine, x);
                raw[i] = make_uint4(0, 0, 0, 0);
                if (x < rows) raw[i] = *reinterpret_cast<const uint4*>(a.query.at + at + lane % kLanes * 16);
            }
#pragma unroll
            for (int i = 0; i < kLanes; ++i)
                *reinterpret_cast<uint4*>(to + swizzled<kTile>(warp_row + i * (32 / kLanes) + lane / kLanes, lane % kLanes)) = raw[i];
            __syncwarp();
            uint32_t tops = 0;
#pragma unroll 4
            for (int i = 0; i < kLanes; ++i) {
                const uint4 x = *reinterpret_cast<const uint4*>(to + swizzled<kTile>(r, i));
                tops = T::max_size(T::max_size(T::max_size(T::max_size(tops, x.x), x.y), x.z), x.w);
            }
            const float2 pair = T::wide(tops);
            const int e = max(int(__float_as_uint(fmaxf(pair.x, pair.y)) >> 23), 27);
            const float up = __uint_as_float(uint32_t(127 + 14 + 127 - e) << 23);
            factor = __uint_as_float(uint32_t(max(e - 14, 1)) << 23) * a.scale;
#pragma unroll 4
            for (int i = 0; i < kLanes; ++i) {
                char* const at = to + swizzled<kTile>(r, i);
                float v[8];
                load8<T>(at, v);
                store_shared(at, pack_half2(v[0] * up, v[1] * up), pack_half2(v[2] * up, v[3] * up),
                             pack_half2(v[4] * up, v[5] * up), pack_half2(v[6] * up, v[7] * up));
            }
            fence_shared();
            __syncwarp();
            if (lane == 0) barrier_arrive(&sh.c.q_full[tile]);
        }

        float m = kLowest, e = kLowest, l = 0.0f;        // as in RowState
        // A step's weights are in tensor memory.
        const auto weighed = [&] {
            __syncwarp();
            tensor_stored();
            fence_before();
            __syncwarp();
            if (lane == 0) barrier_arrive(&sh.c.p_full[tile][turn % 2]);
            ++turn;
        };
        for (int step = begin; step < end; ++step, ++it) {
            if (!warp_wait(&sh.c.s_full[tile][turn % 2], turn / 2 % 2, sh.c)) return;
            fence_after();
            const uint32_t at = scores + turn % 2 * kStep;
            float x[kStep];
            tensor_load(at, x);
            // Never 0, so that a hidden score stays -infinity.
            const float f = fmaxf(factor * sh.c.k_scale[it % kScales], kLeast);
            const float power = sh.c.v_power[it % kScales];
            const uint32_t live = sh.c.live[it % kScales];
            const int see = min(max(seen - step * kStep, 0), kStep);       // columns up to here are seen
            // A weight in the sums is 2^(s f + by), and `share` of it is its part of l. That holds for scores up to
            // `limit`: above it a maximum moves. Where the weights in the sums are too far below l's, or scores so
            // large that their rounding is no small part of a weight, no score is below it.
            const bool odd = power - e < -kFarBelow || large_score(m);
            const float limit = odd ? 2 * kLowest : m + kSlack + fminf(e - power, 0.0f);
            float by = power - e - m, share = exp2_fast(fminf(e - power, kFarBelow));
            tensor_loaded(x);
            const auto seen_bits = [&] {
                uint64_t bits = see == kStep ? ~0ull : (1ull << see) - 1;
#pragma unroll
                for (int i = 0; i < kGranules; ++i)
                    if (!(live >> i & 1)) bits &= ~(0xFFFFull << (kGranule * i));
                return bits;
            };
            if (__any_sync(~0u, see < kStep) || (live & kAllLive) != kAllLive) {
                const uint64_t bits = seen_bits();
#pragma unroll
                for (int i = 0; i < kStep; ++i)
                    if (!(bits >> i & 1)) x[i] = -INFINITY;
            }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < kStep; j += 8)
#pragma unroll
                for (int i = 0; i < 4; ++i) tops[i] = max3(tops[i], x[j + 2 * i], x[j + 2 * i + 1]);
            float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * f;
            if ((live & kApart) || __any_sync(~0u, top > limit)) {
                uint64_t* const summed = step > begin ? &sh.c.o_full[tile][(turn - 1) % 2] : nullptr;
                const uint32_t parity = (turn - 1) / 2 % 2;
                if ((live & kApart) || __any_sync(~0u, odd || large_score(top))) {
                    const bool apart = live & kApart;
                    RowState now{m, e, l};
                    if (!step_alone<D>(now, at, seen_bits(), apart ? sh.c.k_own[it % kScales] : nullptr,
                                       sh.c.v_own[it % kScales], factor, f, power, sums, summed, parity, sh.c))
                        return;
                    m = now.m, e = now.e, l = now.l;
                    weighed();
                    continue;
                }
                // With a larger maximum of the sums comes one of the scores, so that e is no larger than the powers seen.
                const bool lift = top - m + power > e + kSlack;
                if (top > m + (lift ? 0.0f : kSlack)) {      // leaves m + e, and so the sums, as they are
                    const float up = ceilf(top);
                    l *= exp2_fast(m - up);
                    e += m - up, m = up;
                }
                float keep = 1.0f;
                if (lift) {
                    const float up = ceilf(top - m) + power;
                    keep = exp2_fast(e - up);
                    e = up;
                }
                if (summed && __any_sync(~0u, keep != 1.0f) && !rescale<D>(sums, keep, summed, parity, sh.c)) return;
                by = power - e - m, share = exp2_fast(fminf(e - power, kFarBelow));
            }
            float2 some[2] = {};
            const float2 ff = make_float2(f, f), bb = make_float2(by, by);
#pragma unroll
            for (int i = 0; i < kStep; i += 32) {
                uint32_t weights[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    float2 y = fma2(make_float2(x[i + 2 * j], x[i + 2 * j + 1]), ff, bb);
                    y.x = exp2_fast(y.x), y.y = exp2_fast(y.y);
                    some[j % 2] = add2(some[j % 2], y);
                    weights[j] = pack_half2(y.x, y.y);
                }
                __syncwarp();
                tensor_store(at + i / 2, weights);
            }
            some[0] = add2(some[0], some[1]);
            l += (some[0].x + some[0].y) * share;
            weighed();
        }

        if (!warp_wait(&sh.c.o_full[tile][(turn - 1) % 2], (turn - 1) / 2 % 2, sh.c)) return;
        fence_after();
        const bool whole = begin == 0 && end == u.steps;
        const int64_t slot = (2 * int64_t(blockIdx.x) + (begin == 0)) * kUnitRows + tile * kTile + warp_row;
        const bool nans = sh.c.nan_unit[unit % kNanUnits] == int(unit) + 1;
        // A row that sees no token has l = 0, and sums of zero weights that count as zeros.
        const float by = l == 0.0f ? 0.0f : whole ? exp2_fast(e) / l : exp2_fast(e);
        // The queries are done with: their place takes the rows on their way out, 128 bytes of each at a time.
        char* const warp_rows = sh.q[tile] + warp_row * 128;
#pragma unroll 1
        for (int i = 0; i < D; i += 32) {
            float y[32];
            __syncwarp();
            tensor_load(sums + i, y);
            tensor_loaded(y);
#pragma unroll
            for (int j = 0; j < 32; ++j) y[j] *= by;
            if (nans) {
                uint32_t found = 0;
                const int from = max(max(u.first_seen, 0) / kStep, begin) * kStep, to = min(seen, end * kStep);
                for (int t = from; t < to; ++t) {
                    const int64_t block = ints(a.b.table)[u.s * a.b.table_pitch + t / a.c.block_size];
                    if (block < 0 || block >= a.c.blocks) continue;
                    const uint8_t* code = reinterpret_cast<const uint8_t*>(a.c.codes) + a.c.side_pitch +
                                          block * a.c.block_pitch + t % a.c.block_size * a.c.token_pitch +
                                          u.head * a.c.head_pitch + i;
#pragma unroll 1
                    for (int j = 0; j < 32; ++j) found |= uint32_t((code[j] & 0x7F) == 0x7F) << j;
                }
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (found >> j & 1) y[j] = NAN;
            }
            if (whole) {
#pragma unroll
                for (int j = 0; j < 32; j += 8)
                    store_shared(staged(warp_rows, lane, (i % 64 + j) / 8), T::pack(y[j], y[j + 1]),
                                 T::pack(y[j + 2], y[j + 3]), T::pack(y[j + 4], y[j + 5]), T::pack(y[j + 6], y[j + 7]));
                if (i % 64 == 0) continue;
            } else {
#pragma unroll
                for (int j = 0; j < 32; j += 4)
                    store_shared(staged(warp_rows, lane, j / 4), __float_as_uint(y[j]), __float_as_uint(y[j + 1]),
                                 __float_as_uint(y[j + 2]), __float_as_uint(y[j + 3]));
            }
            __syncwarp();
#pragma unroll 2
            for (int j = 0; j < 8; ++j) {
                const int mine = j * 4 + lane / 8;
                const int64_t to = __shfl_sync(~0u, out_row, mine);
                const uint4 piece = *reinterpret_cast<const uint4*>(staged(warp_rows, mine, lane % 8));
                if (mine >= rows) continue;
                char* at = whole ? a.out + (to * D + i - 32) * 2
                                 : reinterpret_cast<char*>(p.parts.sums + (slot + mine) * D + i);
                *reinterpret_cast<uint4*>(at + lane % 8 * 16) = piece;
            }
            __syncwarp();
        }
        if (!whole) {
            if (lane < rows) p.parts.ml[slot + lane] = make_float2(m, l);
            if (begin == 0 && threadIdx.x == 0) {
                const int last = Cut(uint32_t(sh.c.total), gridDim.x).of(uint32_t(u.stop - 1));
                p.parts.units[blockIdx.x] =
                    SharedUnit{u.q.row, u.head, u.first, u.rows, last - int(blockIdx.x) + 1};
            }
        }
        fence_before();                                  // the sums are read before the next unit's are written
        __syncwarp();
        if (lane == 0) barrier_arrive(&sh.c.unit_free[ring]);
        if (final) return;
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kChunkThreads, 1) chunk_kernel(const __grid_constant__ ChunkArgs p) {
    extern __shared__ char raw[];
    auto& sh = *reinterpret_cast<ChunkShared<D>*>(raw + (1024 - shared_address(raw) % 1024) % 1024);
    const AttendArgs& a = p.a;
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32, seqs = a.b.seqs;
    constexpr int kAll = kChunkThreads / 32;
    asm volatile("griddepcontrol.launch_dependents;");
    if (threadIdx.x == 0) p.parts.units[blockIdx.x].parts = 0;

    // All the work (of every sequence, head and row tile, end to end), and where this CTA's begins.
    int64_t mine = 0;
    for (int s = warp; s < seqs; s += kAll) mine += head_cost(a, s);
    if (lane == 0) sh.c.scratch[warp] = mine;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w < kAll; ++w) total += sh.c.scratch[w];
    total *= a.c.kv_heads;
    const Cut cut(uint32_t(total), gridDim.x);
    if (blockIdx.x >= cut.ctas) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const int64_t pos = cut.begin(blockIdx.x), end = cut.begin(blockIdx.x + 1);
    int64_t before = 0;
    for (int base = 0; base < seqs; base += kScanned) {
        for (int s = warp; s < kScanned; s += kAll) {
            const int64_t n = base + s < seqs ? head_cost(a, base + s) : 0;
            if (lane == 0) sh.c.counts[s] = n;
        }
        __syncthreads();
        if (warp == 0) {
            for (int i = 0; i < kScanned; i += 32) {
                const int64_t n = sh.c.counts[i + lane];
                int64_t sum = n * a.c.kv_heads;
#pragma unroll
                for (int k = 1; k < 32; k <<= 1) {
                    const int64_t up = __shfl_up_sync(~0u, sum, k);
                    if (lane >= k) sum += up;
                }
                const int64_t first = before + sum - n * a.c.kv_heads;
                if (n && first <= pos && pos < before + sum) {
                    sh.c.s = base + i + lane;
                    sh.c.head = int((pos - first) / n);
                    sh.c.sought = (pos - first) % n;
                }
                before += __shfl_sync(~0u, sum, 31);
            }
            if (lane == 0) sh.c.scanned = before;
        }
        __syncthreads();
        if (sh.c.scanned > pos) break;
        __syncthreads();
    }
    if (warp == 0) {
        Sequence q;
        chunk_sequence(a, sh.c.s, q);
        int64_t done = 0;
        for (int i = 0; i < row_tiles(a, q); i += 32) {
            const int n = i + lane < row_tiles(a, q) ? kUnitCost + steps_of(a, q, i + lane) : 0;
            int64_t sum = n;
#pragma unroll
            for (int k = 1; k < 32; k <<= 1) {
                const int64_t up = __shfl_up_sync(~0u, sum, k);
                if (lane >= k) sum += up;
            }
            const int64_t first = done + sum - n;
            if (n && first <= sh.c.sought && sh.c.sought < done + sum)
                sh.c.tile = i + lane, sh.c.base = pos - (sh.c.sought - first);
            done += __shfl_sync(~0u, sum, 31);
        }
    }

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            barrier_init(&sh.c.q_full[i], 4);
            barrier_init(&sh.c.s_full[i][0], 1);
            barrier_init(&sh.c.s_full[i][1], 1);
            barrier_init(&sh.c.p_full[i][0], 4);
            barrier_init(&sh.c.p_full[i][1], 4);
            barrier_init(&sh.c.o_full[i][0], 1);
            barrier_init(&sh.c.o_full[i][1], 1);
        }
        for (int i = 0; i < kStages; ++i) {
            barrier_init(&sh.c.k_full[i], kConvertWarps);
            barrier_init(&sh.c.v_full[i], kConvertWarps);
            barrier_init(&sh.c.k_empty[i], 1);
            barrier_init(&sh.c.v_empty[i], 1);
        }
        for (int i = 0; i < kLooked; ++i) {
            barrier_init(&sh.c.looked[i], 1);
            barrier_init(&sh.c.look_free[i], kConvertWarps);
        }
        for (int i = 0; i < kLookedUnits; ++i) {
            barrier_init(&sh.c.unit_looked[i], 1);
            barrier_init(&sh.c.unit_free[i], 9);         // 8 warps of rows, and the issue
        }
        barrier_init(&sh.c.drained, 1);
        sh.c.total = total, sh.c.pos = pos, sh.c.until = end;
        for (int i = 0; i < kNanUnits; ++i) sh.c.nan_unit[i] = 0;
        sh.c.stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssueWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                     ::"r"(shared_address(&sh.c.tensor)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();

    // A part of the work may hold no step: then no role has anything to do.
    Walk w;
    const bool any = w.start(a, sh.c);
    if (!any) {
    } else if (warp < 8) {
        softmax_role<T, D>(p, sh);
    } else if (warp < 8 + kConvertWarps) {
        convert_role<D>(p, sh);
    } else {
        if (warp == kLookWarp) {
            look_role(p, sh.c, w);
        } else if (warp == kIssueWarp) {
            issue_role<D>(sh);
            __syncwarp();
            commit(&sh.c.drained, lane == 0);
            barrier_wait(&sh.c.drained, 0, sh.c, true);
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == kIssueWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh.c.tensor));
    if (threadIdx.x == 0 && sh.c.stop) atomicOr(a.status, KVSNAP_C8_STALLED);
    // These CTAs start as those of the kernel for few rows end, and share nothing with them; what follows needs
    // both kernels' ends.
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- host side ----------------------------------------------------------------------------

// How a call is laid out; the same for its workspace and its launches.
struct Plan {
    StepArgs step;
    bool stepped, chunked;    // whether each kernel runs
    bool split, wide;         // the step kernel's units are cut; more than 8 rows a head
    int step_rows;
    int most_rows;            // that a KV head of a sequence can have
    int64_t ctas, step_ctas, step_units;
    int64_t step_slots, chunk_slots, slots, sum_bytes, bytes;
};

int sm_count() {
    int device = 0, sms = 0;
    check(cudaGetDevice(&device));
    check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    return sms;
}

Plan plan_for(const Cache& c, const Batch& b, int q_heads, int sms) {
    Plan plan{};
    StepArgs& p = plan.step;
    const int group = q_heads / c.kv_heads;
    const int64_t most_rows = int64_t(group) * (b.max_query < b.rows ? b.max_query : b.rows);
    plan.chunked = most_rows > kStepRows;
    plan.most_rows = int(most_rows);
    // With one sequence, the kernel for many rows takes it whatever it holds: one launch, not two (a prompt
    // of 300 tokens 29.3 us, else 32.8).
    // Where no sequence may have rows, it is there to record those that do.
    plan.stepped = !plan.chunked || (group <= kStepRows && b.seqs > 1);
    plan.step_rows = plan.stepped ? kStepRows : 0;
    plan.wide = most_rows > 8;
    // Heads a CTA: up to 8, whose lines of a token lie side by side; but few sequences are spread over CTAs by
    // heads, so that a unit's tokens are cut among fewer CTAs (of 8 heads on 148 SMs, 1 sequence of 8191 tokens
    // takes 17.1 us, with all heads in a CTA 22.4, and 16 sequences 58.0 and 63.6; with a head a CTA 16 sequences
    // take 54.0, 48 of 4000 85.4, and 79.4 by this rule, 64 of 200 31.2 and 18.8).
    p.hc = 1;
    for (int heads = 8; heads > 1; --heads)
        if (c.kv_heads % heads == 0 && int64_t(b.seqs) * (c.kv_heads / heads) >= kSpread) {
            p.hc = heads;
            break;
        }
    p.ts = kWarps / p.hc, p.hg = c.kv_heads / p.hc;
    const int64_t most = (int64_t(b.width) * c.block_size + p.ts * kGranule - 1) / (p.ts * kGranule);
    plan.ctas = sms;
    plan.step_units = int64_t(b.seqs) * p.hg;
    // Cutting the chunks evenly over the CTAs costs a scan of the lengths, merges of parts and a join: as
    // much as 4 chunks in turn, more with more units, up to 20. It saves at most the longest unit's chunks
    // less an even share, taken at half of what the table could hold: the lengths are on the GPU, so over a table
    // much wider than its sequences steps are cut that would be quicker whole. Cut and uncut, in us: 1 sequence
    // of 4000 tokens 16.3 and 25.2; 64 of 300 23.3 and 21.0, of 1000 38.4 and 43.5, of mixed lengths up to 1000
    // 28.1 and 41.6; 128 of 700 47.9 and 40.3; 200 of 700 65.6 and 70.7.
    const int64_t waves = (plan.step_units + sms - 1) / sms;
    const int64_t costs = 4 + (plan.step_units < 96 ? plan.step_units : 96) / 6;
    plan.split = most_rows > 0 && most * (2 * sms * waves - plan.step_units) > costs * 2 * sms;
    plan.step_ctas = plan.split ? plan.ctas : plan.step_units;
    // The two kernels may run at the same time: each has its own part of the workspace.
    plan.step_slots = plan.stepped && plan.split ? 2 * plan.ctas * p.hc * kStepRows : 0;
    plan.chunk_slots = plan.chunked ? 2 * plan.ctas * kUnitRows : 0;
    plan.slots = plan.step_slots + plan.chunk_slots;
    plan.sum_bytes = plan.slots * c.head_dim * int64_t(sizeof(float));
    plan.bytes = plan.slots ? plan.sum_bytes + plan.slots * int64_t(sizeof(float2)) +
                                  2 * plan.ctas * int64_t(sizeof(SharedUnit))
                            : 0;
    return plan;
}

template <typename T, int D, int NT>
void launch_step(const Plan& plan, const StepArgs& p, cudaStream_t stream) {
    const size_t shared = sizeof(StepShared<D, NT>);
    if (plan.split) launch(step_kernel<T, D, NT, true>, dim3(unsigned(plan.step_ctas)), 32 * kWarps, shared, stream, false, p);
    else launch(step_kernel<T, D, NT, false>, dim3(unsigned(plan.step_ctas)), 32 * kWarps, shared, stream, false, p);
}

template <typename T, int D>
void launch_attend(const Plan& plan, const AttendArgs& a, char* workspace, cudaStream_t stream) {
    const unsigned ctas = unsigned(plan.ctas);
    const Parts of_steps{reinterpret_cast<float*>(workspace), reinterpret_cast<float2*>(workspace + plan.sum_bytes),
                   reinterpret_cast<SharedUnit*>(workspace + plan.sum_bytes + plan.slots * int64_t(sizeof(float2))),
                   plan.step.hc, kStepRows, plan.wide ? kStepRows : plan.most_rows};
    const Parts of_chunks{of_steps.sums + plan.step_slots * D, of_steps.ml + plan.step_slots, of_steps.units + ctas,
                          1, kUnitRows, plan.most_rows < kUnitRows ? plan.most_rows : kUnitRows};
    if (plan.stepped) {
        StepArgs p = plan.step;
        p.a = a, p.parts = of_steps;
        if (plan.wide) launch_step<T, D, 2>(plan, p, stream);
        else launch_step<T, D, 1>(plan, p, stream);
    }
    // Without a wait between the two, batches of steps and chunks gain 6 % (16 sequences of up to 4000 tokens, with
    // 1 and 9 new ones by turns, 64.5 us; one kernel after the other 68.4).
    if (plan.chunked)
        launch(chunk_kernel<T, D>, dim3(ctas), kChunkThreads, sizeof(ChunkShared<D>) + 1024, stream, plan.stepped,
               ChunkArgs{a, of_chunks});
    if (!plan.slots) return;
    // Few units have many parts each, and a CTA joins a row (8 units' 8191 tokens 17.1 us, a warp a row 18.9);
    // many have few, as chunks do, and a warp does (chunks of 128 tokens in 24 sequences 185 us, a CTA a row 269).
    const bool wide = !plan.chunked && plan.step_units * 8 <= plan.ctas;
    const auto high = [&](const Parts& p) {
        const unsigned rows = unsigned(p.heads * p.used_rows);
        return wide ? rows : (rows + kJoinWarps - 1) / kJoinWarps;
    };
    const unsigned joined = plan.step_slots ? ctas : 0, step_high = high(of_steps), chunk_high = high(of_chunks);
    const dim3 grid(joined * step_high + (plan.chunked ? ctas * chunk_high : 0));
    launch(wide ? join_kernel<T, D, true> : join_kernel<T, D, false>, grid, 32 * kJoinWarps, 0, stream, true, a, of_steps,
           joined, step_high, of_chunks, chunk_high);
}

void check_attend(const Cache* cache, const Batch* batch, int q_heads) {
    check_cache(cache);
    check_batch(batch, cache);
    require(q_heads > 0 && q_heads % cache->kv_heads == 0, "query heads must be a multiple of the KV heads");
    require(int64_t(batch->seqs) * cache->kv_heads < (1LL << 30) && int64_t(batch->rows) * q_heads < (1LL << 30),
            "too many sequences or rows for one attention");
    // All the work of a call is counted in 32 bits: granules of each head, steps of each 256 rows and head.
    const double granules = double(batch->width) * cache->block_size / kGranule + 1;
    const double units = double(batch->rows) * (q_heads / cache->kv_heads) / kUnitRows + batch->seqs;
    require(batch->seqs * (granules + kStepUnitCost) * cache->kv_heads < 2147483648.0 &&
                units * cache->kv_heads * (granules * kGranule / kStep + kUnitCost + 1) < 2147483648.0,
            "too much work for one attention");
}

}  // namespace

extern "C" int kvsnap_c8_attend_workspace(const kvsnap_c8_cache* cache, const kvsnap_c8_batch* batch, int q_heads,
                                          size_t* bytes) {
    return on_device(cache ? cache->device : 0, [&] {
        check_attend(cache, batch, q_heads);
        require(bytes, "the workspace's size needs a place");
        *bytes = 0;
        return batch->rows && batch->seqs;
    }, [&] {
        *bytes = size_t(plan_for(*cache, *batch, q_heads, sm_count()).bytes);
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
        require(scale >= 0.0f && scale <= 3.402823466e38f, "the scores' scale must be finite and not negative");
        return true;
    }, [&] {
        const Plan plan = plan_for(*cache, *batch, q_heads, sm_count());
        require(!plan.bytes || (workspace && int64_t(workspace_bytes) >= plan.bytes &&
                                aligned(reinterpret_cast<intptr_t>(workspace))),
                "the attention's workspace is too small or not 16-byte aligned");
        const AttendArgs a{*cache, *batch, {static_cast<const char*>(query), query_token, query_head},
                           static_cast<char*>(out), q_heads, q_heads / cache->kv_heads, plan.step_rows,
                           scale * 1.4426950408889634f, status};
        by_type(type, cache->head_dim, [&](auto t, auto d) {
            launch_attend<decltype(t), decltype(d)::value>(plan, a, static_cast<char*>(workspace),
                                                           reinterpret_cast<cudaStream_t>(stream));
        });
    });
}
