// sm_100a kernels that fill the 8-bit paged KV cache: append with rotation, and
// conversion of blocks between 16-bit caches and this one. The format is
// described in cache8.cuh; attention over it is attend8.cu.
#include "cache8.cuh"

namespace {

// ---- append ------------------------------------------------------------------------

struct AppendArgs {
    Cache c;
    Batch b;
    Rows key, value, query;
    char* query_out;
    const float2* rotary;     // [positions][rotary_dim / 2] (cos, sin)
    int64_t positions;
    int rotary_dim, q_heads;  // 0: no rotation; no queries
    uint32_t* status;
};

// Where one unit of an append lies: a page of a sequence and the new rows in it.
struct PageRun {
    int seq, page;            // the sequence, and the page's place in its table row
    int first, count;         // slots [first, first + count) are new
    int row;                  // token row of slot `first`
};

// Unit u's page, its positions in 32 bits (a table row holds at most 2^30 tokens). Sequence s's units start at start[s] / N + 2 s, which leaves each
// sequence room for the pages that its rows can touch ((rows - 2) / N + 2), whatever
// slot they start in, so a unit finds its sequence by bisection with no scan over
// the batch. With one row a sequence (SINGLE) unit u is sequence u.
template <bool SINGLE>
__device__ __forceinline__ bool find_page(const Batch& b, int n, int64_t u, PageRun& run, uint32_t* status) {
    const int32_t* start = ints(b.start);
    int s = int(u), k = 0;
    if (!SINGLE) {
        int lo = 0, hi = b.seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (int64_t(max(start[mid], 0)) / n + 2 * int64_t(mid) <= u) lo = mid; else hi = mid - 1;
        }
        s = lo;
        const int64_t past = u - (int64_t(max(start[s], 0)) / n + 2 * int64_t(s));
        if (past < 0 || past >= b.width) return false;
        k = int(past);
    }
    const int from = start[s], to = start[s + 1], length = ints(b.lengths)[s];
    if (from >= to || length <= 0) return false;
    if (from < 0 || to > b.rows || to - from > b.max_query || int64_t(length) > int64_t(b.width) * n) {
        atomicOr(status, KVSNAP_C8_BAD_LENGTH);
        return false;
    }
    const int held = max(length - (to - from), 0);        // tokens before the new ones
    run.seq = s;
    run.page = held / n + k;
    const int base = run.page * n;
    if (base >= length) return false;
    run.first = k ? 0 : held - int(base);
    run.count = min(n, int(length - base)) - run.first;
    run.row = to - (length - int(base)) + run.first;
    return true;
}

// The page's rows that the rotary table has angles for; false where there are none. The others are left out and
// recorded.
__device__ __forceinline__ bool within_table(const AppendArgs& a, PageRun& run) {
    const int64_t left = a.positions - (int64_t(run.page) * a.c.block_size + run.first);
    if (!a.rotary_dim || left >= run.count) return true;
    if (threadIdx.x == 0) atomicOr(a.status, KVSNAP_C8_BAD_POSITION);
    run.count = int(max(left, int64_t(0)));
    return run.count > 0;
}

// A lane's 8 elements of a row of rotated heads: 4 from `low` on and 4 from `high` on, 4 whole pairs, so that
// nothing passes between lanes and a row's angles are read once: of a row of 16 lanes each reads 8 bytes
// of two lines, and 32 bytes of angles. Elements from rotary_dim on, and interleaved pairs, lie together.
struct Place {
    int low, high, pair;
    bool turned;

    __device__ __forceinline__ Place(int lane, int rotary_dim, bool interleaved) : pair(4 * lane) {
        turned = 8 * lane < rotary_dim;
        const bool apart = turned && !interleaved;
        low = apart ? 4 * lane : 8 * lane, high = apart ? rotary_dim / 2 + 4 * lane : 8 * lane + 4;
    }
};

// (cos, sin) of a lane's 4 pairs.
struct Turn {
    uint4 x[2];
};

__device__ __forceinline__ void fetch_turn(Turn& turn, const AppendArgs& a, int64_t position, const Place& at,
                                           bool there) {
    // Lanes past the page's rows have positions too, for which nothing is fetched. They are held within the table:
    // without that the compiler's code for an 8k prompt takes 53.3 us, so 52.3.
    const float2* from = a.rotary + min(position, a.positions - 1) * (a.rotary_dim / 2) + at.pair;
#pragma unroll
    for (int i = 0; i < 2; ++i) turn.x[i] = fetch16(reinterpret_cast<const char*>(from + 2 * i), there && at.turned);
}

__device__ __forceinline__ uint4 fetch_place(const char* row, const Place& at, bool there) {
    const uint2 low = fetch8(row + 2 * at.low, there), high = fetch8(row + 2 * at.high, there);
    return make_uint4(low.x, low.y, high.x, high.y);
}

template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void turn8(const uint4& raw, const Turn& turn, const Place& at, float (&v)[8]) {
    widen8<T>(raw, v);
    if (!at.turned) return;
    const float* cs = reinterpret_cast<const float*>(turn.x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float& p = v[INTERLEAVED ? 2 * i : i];
        float& q = v[INTERLEAVED ? 2 * i + 1 : 4 + i];
        const float x = p, y = q;
        p = x * cs[2 * i] - y * cs[2 * i + 1];
        q = y * cs[2 * i] + x * cs[2 * i + 1];
    }
}

constexpr int kHeld = 8;      // row groups of a page that a warp keeps in registers, as they come

// The largest finite size among a warp's rows: of the 16-bit words as they are, and where that is no
// finite number, once more without those that are not.
template <typename T, int N>
__device__ __forceinline__ float largest(const uint4 (&raw)[N]) {
    uint32_t tops = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
        tops = T::max_size(T::max_size(T::max_size(T::max_size(tops, raw[i].x), raw[i].y), raw[i].z), raw[i].w);
    const float2 pair = T::wide(tops);
    float top = warp_max(fmaxf(pair.x, pair.y));
    if (top > 3.402823466e38f) {
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float v[8];
            widen8<T>(raw[i], v);
            top = max8(v, top);
        }
        top = warp_max(top);
    }
    return top;
}

template <int N>
__device__ __forceinline__ float largest(const float (&v)[N][8]) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(v[i][k]));        // of a number and NaN, the number
    top = warp_max(top);
    if (top > 3.402823466e38f) {
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) top = max8(v[i], top);
        top = warp_max(top);
    }
    return top;
}

// Append: one CTA takes page blockIdx.x and 8 key or value heads, a warp each, or 8 query heads. A row is
// D / 8 lanes of 8 elements, so a warp takes 256 / D rows at a time. Turned: (x cos - y sin, y cos + x sin) of
// each pair, in 32 bits. Bound by memory, so all loads of a warp are issued together, predicated. Keys and
// values hold a page's rows in registers from their fetch to their codes, as the scale needs all rows
// first (128 registers a thread); queries are turned as they come (64). An 8k prompt of 32 and 8 heads of
// 128: the queries' 134 MB in 20 us, 6.6 TB/s; the keys' and values' 50 MB in 18 us, bound by the way of the
// loads of 16 warps an SM (turned twice from what had come, for the scale and for the codes, 28 us).

// 8 query heads of a page's rows from 8 y on, of which each warp takes some rows (of a single row, a head). A
// row's angles are fetched once for the 8.
template <typename T, int D, bool SINGLE, bool INTERLEAVED>
__device__ __forceinline__ void turn_queries(const AppendArgs& a, int y) {
    constexpr int kLanes = D / 8, kRows = 32 / kLanes, kTogether = SINGLE ? 1 : 8;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, n = a.c.block_size;
    PageRun run;
    if (!find_page<SINGLE>(a.b, n, blockIdx.x, run, a.status) || !within_table(a, run)) return;
    const int sub = lane / kLanes, end = run.first + run.count;
    const int base = run.page * n;                               // position of the page's slot 0
    const Place place(lane % kLanes, a.rotary_dim, INTERLEAVED);
    const int head = y * 8 + (SINGLE ? warp : 0), heads = min(SINGLE ? 1 : 8, a.q_heads - head);
    for (int first = run.first + (SINGLE ? 0 : warp * kRows); first < end; first += 8 * kRows) {
        const int r = first + sub;
        const int64_t row = run.row + (r - run.first);
        const char* from = a.query.at + row * a.query.token + head * a.query.head;
        char* to = a.query_out + (row * a.q_heads + head) * (2 * D);
        Turn turn;
        fetch_turn(turn, a, base + r, place, r < end);
        uint4 raw[kTogether];
#pragma unroll
        for (int i = 0; i < kTogether; ++i) raw[i] = fetch_place(from + i * a.query.head, place, r < end && i < heads);
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
            float v[8];
            turn8<T, INTERLEAVED>(raw[i], turn, place, v);
            if (r < end && i < heads) {
                char* const out = to + i * (2 * D);
                *reinterpret_cast<uint2*>(out + 2 * place.low) = make_uint2(T::pack(v[0], v[1]), T::pack(v[2], v[3]));
                *reinterpret_cast<uint2*>(out + 2 * place.high) = make_uint2(T::pack(v[4], v[5]), T::pack(v[6], v[7]));
            }
        }
    }
}

// Key and value heads from 8 y on: the values' behind the keys'.
template <typename T, int D, bool SINGLE, bool INTERLEAVED>
__device__ __forceinline__ void append_rows(const AppendArgs& a, int y) {
    constexpr int kLanes = D / 8, kRows = 32 / kLanes, kHeld = SINGLE ? 1 : ::kHeld;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, n = a.c.block_size, slot = y * 8 + warp;
    if (slot >= 2 * a.c.kv_heads) return;
    PageRun run;
    if (!find_page<SINGLE>(a.b, n, blockIdx.x, run, a.status) || !within_table(a, run)) return;
    const int sub = lane / kLanes, at = lane % kLanes * 8, end = run.first + run.count;
    const int base = run.page * n;                               // position of the page's slot 0
    const Place place(lane % kLanes, a.rotary_dim, INTERLEAVED);

    const int side = slot / a.c.kv_heads, head = slot % a.c.kv_heads;
    const int64_t block = ints(a.b.table)[run.seq * a.b.table_pitch + run.page];
    if (block < 0 || block >= a.c.blocks) {
        if (lane == 0) atomicOr(a.status, KVSNAP_DP_BAD_BLOCK);
        return;
    }
    char* codes = reinterpret_cast<char*>(a.c.codes) + side * a.c.side_pitch + block * a.c.block_pitch +
                  head * a.c.head_pitch;
    float* scale_at = reinterpret_cast<float*>(a.c.scales) + (block * 2 + side) * a.c.kv_heads + head;
    const Rows& from = side ? a.value : a.key;
    const char* rows = from.at + head * from.head + (run.row - run.first) * from.token;
    const float held = run.first ? *scale_at : 0.0f;
    float scale = 0.0f, by = 0.0f;
    const auto sized = [&](float top) { scale = fmaxf(held, needed_scale(top)), by = inverse(scale); };
    // The largest size of all rows, then their codes; rows too many to hold are fetched twice.
    const int together = kHeld * kRows, passes = run.count > together ? 2 : 1;
    float top = 0.0f;
    if (side == 0 && a.rotary_dim) {
#pragma unroll 1
        for (int pass = 0; pass < passes; ++pass)
            for (int first = run.first; first < end; first += together) {
                float v[kHeld][8];
                uint4 raw[kHeld];
                constexpr int kTurns = SINGLE ? 1 : kHeld - 2;      // on their way together: all would be spilled
                Turn turn[kTurns];
#pragma unroll
                for (int i = 0; i < kHeld; ++i) {
                    const int r = first + i * kRows + sub;
                    if (i < kTurns) fetch_turn(turn[i], a, base + r, place, r < end);
                    raw[i] = fetch_place(rows + r * from.token, place, r < end);
                }
#pragma unroll
                for (int i = 0; i < kHeld; ++i) {
                    turn8<T, INTERLEAVED>(raw[i], turn[i % kTurns], place, v[i]);
                    const int next = i + kTurns, r = first + next * kRows + sub;
                    if (next < kHeld) fetch_turn(turn[i], a, base + r, place, r < end);
                }
                if (pass == 0) top = fmaxf(top, largest(v));
                if (pass + 1 < passes) continue;
                sized(top);
#pragma unroll
                for (int i = 0; i < kHeld; ++i) {
                    const int r = first + i * kRows + sub;
                    const uint2 both = codes_of(v[i], by);
                    if (r < end) {
                        *reinterpret_cast<uint32_t*>(codes + r * a.c.token_pitch + place.low) = both.x;
                        *reinterpret_cast<uint32_t*>(codes + r * a.c.token_pitch + place.high) = both.y;
                    }
                }
            }
    } else {
#pragma unroll 1
        for (int pass = 0; pass < passes; ++pass)
            for (int first = run.first; first < end; first += together) {
                uint4 raw[kHeld];
#pragma unroll
                for (int i = 0; i < kHeld; ++i) {
                    const int r = first + i * kRows + sub;
                    raw[i] = fetch16(rows + r * from.token + 2 * at, r < end);
                }
                if (pass == 0) top = fmaxf(top, largest<T>(raw));
                if (pass + 1 < passes) continue;
                sized(top);
#pragma unroll
                for (int i = 0; i < kHeld; ++i) {
                    const int r = first + i * kRows + sub;
                    float v[8];
                    widen8<T>(raw[i], v);
                    if (r < end) store_codes(codes + r * a.c.token_pitch + at, v, by);
                }
            }
    }
    if (!run.first || scale > held) {
        for (int r = sub; r < run.first; r += kRows) {                 // older tokens, at the grown scale
            float v[8];
            load_codes(codes + r * a.c.token_pitch + at, held, v);
            store_codes(codes + r * a.c.token_pitch + at, v, by);
        }
        __syncwarp();
        if (lane == 0) *scale_at = scale;
    }
}

// One row a sequence: a token of each of 64 sequences takes 4.5 us, which is a launch and two fetches, one
// after the other, with nothing in the caches.
template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 4) append_one_kernel(const __grid_constant__ AppendArgs a) {
    const int kv_ctas = (2 * a.c.kv_heads + 7) / 8;
    if (blockIdx.y < kv_ctas) append_rows<T, D, true, INTERLEAVED>(a, blockIdx.y);
    else turn_queries<T, D, true, INTERLEAVED>(a, blockIdx.y - kv_ctas);
}

// The queries too where the grid has CTAs for them; otherwise they are turn_kernel's, whose CTAs start as
// these end.
template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 2) append_kernel(const __grid_constant__ AppendArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    const int kv_ctas = (2 * a.c.kv_heads + 7) / 8;
    if (blockIdx.y < kv_ctas) append_rows<T, D, false, INTERLEAVED>(a, blockIdx.y);
    else turn_queries<T, D, false, INTERLEAVED>(a, blockIdx.y - kv_ctas);
}

template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 4) turn_kernel(const __grid_constant__ AppendArgs a) {
    turn_queries<T, D, false, INTERLEAVED>(a, blockIdx.y);
    asm volatile("griddepcontrol.wait;" ::: "memory");       // what follows in the stream needs both kernels' ends
}

// ---- conversion ----------------------------------------------------------------------

struct ConvertArgs {
    const kvsnap_c8_pair* pairs;
    const int64_t *ids, *wide_ids;
    int64_t n, valid;
    int layers, block_size, kv_heads;
    uint32_t* status;
};

// One warp: one layer, block, side and head. Grid: (block and head, layer and side).
struct ConvertUnit {
    char *codes, *wide;
    float* scale;
    int64_t token, wide_token;
    int rows;                 // token slots that hold tokens
};

__device__ __forceinline__ bool convert_unit(const ConvertArgs& a, ConvertUnit& unit) {
    const uint32_t u = blockIdx.x * 8 + threadIdx.x / 32;
    const int64_t i = u / a.kv_heads;
    const int head = u % a.kv_heads, side = blockIdx.y & 1;
    if (i >= a.n) return false;
    const kvsnap_c8_pair& p = a.pairs[blockIdx.y / 2];
    const int64_t block = a.ids[i], from = a.wide_ids[i];
    if (block < 0 || block >= p.blocks || from < 0 || from >= p.wide_blocks) {
        if (threadIdx.x % 32 == 0) atomicOr(a.status, KVSNAP_DP_BAD_BLOCK);
        return false;
    }
    unit.codes = reinterpret_cast<char*>(p.codes) + side * p.side_pitch + block * p.block_pitch + head * p.head_pitch;
    unit.wide = reinterpret_cast<char*>(p.wide) + side * p.wide_side + from * p.wide_block + head * p.wide_head;
    unit.scale = reinterpret_cast<float*>(p.scales) + (block * 2 + side) * a.kv_heads + head;
    unit.token = p.token_pitch, unit.wide_token = p.wide_token;
    const int64_t left = a.valid < 0 ? a.block_size : a.valid - i * a.block_size;
    unit.rows = int(left < 0 ? 0 : left > a.block_size ? a.block_size : left);
    return true;
}

// Bound by memory: a warp holds a page's head as it comes (32 registers), so that four CTAs an SM keep
// 128 KB of loads on their way. 8192 tokens of 36 layers of 8 heads of 128, 1.8 GB, take 274 us: 6.6 TB/s,
// the rate of a plain copy.
template <typename T, int D>
__global__ void __launch_bounds__(256, 4) compress_kernel(const __grid_constant__ ConvertArgs a) {
    constexpr int kLanes = D / 8, kRows = 32 / kLanes;
    const int lane = threadIdx.x % 32, sub = lane / kLanes, at = lane % kLanes * 8;
    ConvertUnit unit;
    if (!convert_unit(a, unit)) return;
    const char* from = unit.wide + 2 * at;
    uint4 raw[kHeld];
    const auto fetch = [&](int first) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int r = first + i * kRows + sub;
            raw[i] = fetch16(from + r * unit.wide_token, r < unit.rows);
        }
    };
    float top = 0.0f;
    for (int first = kHeld * kRows; first < unit.rows; first += kHeld * kRows) {     // rows too many to hold
        fetch(first);
        top = fmaxf(top, largest<T>(raw));
    }
    fetch(0);
    const float scale = needed_scale(fmaxf(top, largest<T>(raw))), by = inverse(scale);
    for (int first = 0; first < a.block_size; first += kHeld * kRows) {
        if (first) fetch(first);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int r = first + i * kRows + sub;
            float v[8];
            widen8<T>(raw[i], v);
            if (r < a.block_size) store_codes(unit.codes + r * unit.token + at, v, by);
        }
    }
    if (lane == 0) *unit.scale = scale;
}

// 8 codes a lane, so that a store instruction's 16 bytes a lane are whole lines (16 codes a lane wrote
// every other 16 bytes: 5.1 TB/s where this reaches 6.7, 1.8 GB in 269 us). Bound by memory.
template <typename T, int D>
__global__ void __launch_bounds__(256, 4) expand_kernel(const __grid_constant__ ConvertArgs a) {
    constexpr int kLanes = D / 8, kRows = 32 / kLanes, kSteps = kGranule / kRows;
    const int lane = threadIdx.x % 32, sub = lane / kLanes, at = lane % kLanes * 8;
    ConvertUnit unit;
    if (!convert_unit(a, unit)) return;
    const float scale = *unit.scale;
    for (int first = sub; first < a.block_size; first += kGranule) {
        uint2 raw[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) raw[i] = fetch8(unit.codes + (first + i * kRows) * unit.token + at, true);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            float v[8];
            widen_codes(raw[i], scale, v);
            char* to = unit.wide + (first + i * kRows) * unit.wide_token + 2 * at;
            const uint4 x = make_uint4(T::pack(v[0], v[1]), T::pack(v[2], v[3]), T::pack(v[4], v[5]), T::pack(v[6], v[7]));
            *reinterpret_cast<uint4*>(to) = x;
        }
    }
}

}  // namespace

extern "C" int kvsnap_c8_append(const kvsnap_c8_cache* cache, const kvsnap_c8_batch* batch, int type, const void* key,
                                int64_t key_token, int64_t key_head, const void* value, int64_t value_token,
                                int64_t value_head, const void* query, int64_t query_token, int64_t query_head,
                                int q_heads, void* query_out, const float* rotary, int64_t positions, int rotary_dim,
                                int interleaved, uint32_t* status, uintptr_t stream) {
    return on_device(cache ? cache->device : 0, [&] {
        check_cache(cache);
        check_batch(batch, cache);
        require(status, "the append needs a status word");
        if (!batch->rows || !batch->seqs) return false;
        check_rows(key, key_token, key_head);
        check_rows(value, value_token, value_head);
        if (query) check_rows(query, query_token, query_head);
        check_type(type);
        require(!query || (q_heads > 0 && query_out), "the rotated query needs heads and an output");
        require(!rotary || (rotary_dim > 0 && rotary_dim % 16 == 0 && rotary_dim <= cache->head_dim && positions > 0),
                "rotary_dim must be a multiple of 16 up to head_dim");
        require(batch->rows / cache->block_size + 2LL * batch->seqs < (1LL << 31), "too many rows for one append");
        return true;
    }, [&] {
        const AppendArgs a{*cache, *batch, {static_cast<const char*>(key), key_token, key_head},
                           {static_cast<const char*>(value), value_token, value_head},
                           {static_cast<const char*>(query), query_token, query_head},
                           static_cast<char*>(query_out), reinterpret_cast<const float2*>(rotary), positions,
                           rotary ? rotary_dim : 0, query ? q_heads : 0, status};
        const bool single = batch->max_query <= 1;
        const int64_t units = single ? batch->seqs : batch->rows / cache->block_size + 2LL * batch->seqs;
        const unsigned kv_ctas = unsigned(2 * cache->kv_heads + 7) / 8, q_ctas = unsigned(a.q_heads + 7) / 8;
        by_type(type, cache->head_dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int D = decltype(d)::value;
            const auto s = reinterpret_cast<cudaStream_t>(stream);
            const auto run = [&](auto kernel, unsigned high, bool beside) {
                launch(kernel, dim3(unsigned(units), high), 256, 0, s, beside, a);
            };
            if (single) {
                run(interleaved ? append_one_kernel<T, D, true> : append_one_kernel<T, D, false>, kv_ctas + q_ctas, false);
                return;
            }
            // Queries in a launch of their own are worth it from three full waves of the GPU's 148 SMs on; below that
            // the launch costs more. Of 32 and 8 heads of 128, together and apart, in us (a call; in a graph): 1500
            // tokens, 576 CTAs, 11.9 and 14.2 (9.2, 10.1); 2600, 984 CTAs, 16.9 and 17.0 (14.1, 14.4); 4000,
            // 1512 CTAs, 23.0 and 21.0 (20.1, 18.8); 8192, 3084 CTAs, 41.6 and 39.9 (39.5, 37.5).
            const bool apart = q_ctas && units * (kv_ctas + q_ctas) > 1000;
            run(interleaved ? append_kernel<T, D, true> : append_kernel<T, D, false>, kv_ctas + (apart ? 0 : q_ctas), false);
            if (apart) run(interleaved ? turn_kernel<T, D, true> : turn_kernel<T, D, false>, q_ctas, true);
        });
    });
}

namespace {

template <bool EXPAND>
int convert(const kvsnap_c8_pair* pairs, int layers, int block_size, int kv_heads, int head_dim, int type,
            const int64_t* ids, const int64_t* wide_ids, int64_t n, int64_t valid, uint32_t* status, int device,
            uintptr_t stream) {
    return on_device(device, [&] {
        require(layers >= 0 && n >= 0 && status, "invalid conversion");
        if (!layers || !n) return false;
        require(pairs && ids && wide_ids, "invalid conversion");
        check_type(type);
        require(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");
        require(block_size > 0 && block_size % 16 == 0 && kv_heads > 0, "block_size must be a multiple of 16");
        require(n < (1LL << 31) && n * kv_heads < (1LL << 31) && layers <= 32767, "too many blocks for one conversion");
        return true;
    }, [&] {
        const ConvertArgs a{pairs, ids, wide_ids, n, valid, layers, block_size, kv_heads, status};
        const dim3 grid(unsigned((n * kv_heads + 7) / 8), unsigned(2 * layers));
        by_type(type, head_dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int D = decltype(d)::value;
            const auto s = reinterpret_cast<cudaStream_t>(stream);
            if (EXPAND) launch(expand_kernel<T, D>, grid, 256, 0, s, false, a);
            else launch(compress_kernel<T, D>, grid, 256, 0, s, false, a);
        });
    });
}

}  // namespace

extern "C" int kvsnap_c8_compress(const kvsnap_c8_pair* pairs, int layers, int block_size, int kv_heads, int head_dim,
                                  int type, const int64_t* wide_ids, const int64_t* ids, int64_t n,
                                  int64_t valid_tokens, uint32_t* status, int device, uintptr_t stream) {
    return convert<false>(pairs, layers, block_size, kv_heads, head_dim, type, ids, wide_ids, n, valid_tokens, status,
                          device, stream);
}

extern "C" int kvsnap_c8_expand(const kvsnap_c8_pair* pairs, int layers, int block_size, int kv_heads, int head_dim,
                                int type, const int64_t* ids, const int64_t* wide_ids, int64_t n, uint32_t* status,
                                int device, uintptr_t stream) {
    return convert<true>(pairs, layers, block_size, kv_heads, head_dim, type, ids, wide_ids, n, -1, status, device,
                         stream);
}
