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
    const float2* rotary;     // [positions][rotary_dim / 2] (cos, sin); NULL: no rotation
    int64_t positions;
    int rotary_dim, q_heads;
    uint32_t* status;
};

// Where one unit of an append lies: a page of a sequence and the new rows in it.
struct PageRun {
    int seq, page;            // the sequence, and the page's place in its table row
    int first, count;         // slots [first, first + count) are new
    int row;                  // token row of slot `first`
};

// Unit u's page. Sequence s's units start at start[s] / N + 2 s, which leaves each
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
        if (past < 0) return false;
        k = int(past);
    }
    const int from = start[s], to = start[s + 1], length = ints(b.lengths)[s];
    if (from >= to || length <= 0) return false;
    if (from < 0 || to > b.rows || (SINGLE && to - from > 1) || int64_t(length) > int64_t(b.width) * n) {
        atomicOr(status, KVSNAP_C8_BAD_LENGTH);
        return false;
    }
    const int held = max(length - (to - from), 0);        // tokens before the new ones
    run.seq = s;
    run.page = held / n + k;
    const int64_t base = int64_t(run.page) * n;
    if (base >= length) return false;
    run.first = k ? 0 : held - int(base);
    run.count = min(n, int(length - base)) - run.first;
    run.row = to - (length - int(base)) + run.first;
    return true;
}

// The rotation of 8 consecutive elements [at, at + 8) of a head, from its row in memory.
template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void load_rotated(const char* row, int at, const float2* turn, int rotary_dim,
                                             float (&v)[8]) {
    load8<T>(row + 2 * at, v);
    if (!turn || at >= rotary_dim) return;
    if (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = turn[at / 2 + i];
            const float a = v[2 * i], b = v[2 * i + 1];
            v[2 * i] = a * t.x - b * t.y;
            v[2 * i + 1] = b * t.x + a * t.y;
        }
    } else {
        const int half = rotary_dim / 2;
        const bool low = at < half;
        const int pair = low ? at : at - half;
        float w[8];
        load8<T>(row + 2 * (low ? at + half : at - half), w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 t = turn[pair + i];
            v[i] = low ? v[i] * t.x - w[i] * t.y : v[i] * t.x + w[i] * t.y;
        }
    }
}

constexpr int kHeld = 8;      // row groups of a page that a warp keeps in registers (64 values a lane)

// One warp: one page of one key or value head, or its query rows of one query head.
// A row is D / 8 lanes of 8 elements, so a warp takes 256 / D rows a step.
template <typename T, int D, bool SINGLE, bool INTERLEAVED>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int kLanes = D / 8, kRows = 32 / kLanes;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, n = a.c.block_size;
    const int slot = blockIdx.y * 8 + warp;
    if (slot >= 2 * a.c.kv_heads + a.q_heads) return;
    PageRun run;
    if (!find_page<SINGLE>(a.b, n, blockIdx.x, run, a.status)) return;
    const int sub = lane / kLanes, at = lane % kLanes * 8;
    const int64_t base = int64_t(run.page) * n;                        // position of the page's slot 0

    const auto turn = [&](int r) -> const float2* {                    // row r of the page
        if (!a.rotary) return nullptr;
        int64_t p = base + r;
        if (p >= a.positions) {
            atomicOr(a.status, KVSNAP_C8_BAD_POSITION);
            p = a.positions - 1;
        }
        return a.rotary + p * (a.rotary_dim / 2);
    };

    if (slot >= 2 * a.c.kv_heads) {
        const int head = slot - 2 * a.c.kv_heads;
        for (int r = run.first + sub; r < run.first + run.count; r += kRows) {
            const int64_t row = run.row + (r - run.first);
            float v[8];
            load_rotated<T, INTERLEAVED>(a.query.at + row * a.query.token + head * a.query.head, at, turn(r),
                                         a.rotary_dim, v);
            store8<T>(a.query_out + ((row * a.q_heads + head) * D + at) * 2, v);
        }
        return;
    }

    const int side = slot / a.c.kv_heads, head = slot % a.c.kv_heads;
    const int64_t block = ints(a.b.table)[run.seq * a.b.table_pitch + run.page];
    if (block < 0 || block >= a.c.blocks) {
        if (lane == 0) atomicOr(a.status, KVSNAP_DP_BAD_BLOCK);
        return;
    }
    char* codes = reinterpret_cast<char*>(a.c.codes) + side * a.c.side_pitch + block * a.c.block_pitch +
                  head * a.c.head_pitch + at;
    float* scale_at = reinterpret_cast<float*>(a.c.scales) + (block * 2 + side) * a.c.kv_heads + head;
    const Rows& from = side ? a.value : a.key;
    const char* rows = from.at + head * from.head;
    const auto fetch = [&](int r, float (&v)[8]) {
        const char* row = rows + (run.row + (r - run.first)) * from.token;
        if (side) load8<T>(row + 2 * at, v);
        else load_rotated<T, INTERLEAVED>(row, at, turn(r), a.rotary_dim, v);
    };

    const int end = run.first + run.count;
    float kept[kHeld][8], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int r = run.first + i * kRows + sub;
        if (r < end) {
            fetch(r, kept[i]);
            amax = max8(kept[i], amax);
        }
    }
    for (int r = run.first + kHeld * kRows + sub; r < end; r += kRows) {
        float v[8];
        fetch(r, v);
        amax = max8(v, amax);
    }
    const float held = run.first ? *scale_at : 0.0f;
    const float scale = fmaxf(held, needed_scale(warp_max(amax)));
    const float by = inverse(scale);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int r = run.first + i * kRows + sub;
        if (r < end) store_codes(codes + r * a.c.token_pitch, kept[i], by);
    }
    for (int r = run.first + kHeld * kRows + sub; r < end; r += kRows) {
        float v[8];
        fetch(r, v);
        store_codes(codes + r * a.c.token_pitch, v, by);
    }
    if (!run.first || scale > held) {
        for (int r = sub; r < run.first; r += kRows) {                 // older tokens, at the grown scale
            float v[8];
            load_codes(codes + r * a.c.token_pitch, held, v);
            store_codes(codes + r * a.c.token_pitch, v, by);
        }
        __syncwarp();
        if (lane == 0) *scale_at = scale;
    }
}

// ---- conversion ----------------------------------------------------------------------

struct ConvertArgs {
    const kvsnap_c8_pair* pairs;
    const int64_t *ids, *wide_ids;
    int64_t n, valid;
    int layers, block_size, kv_heads;
    uint32_t* status;
};

// One warp: one layer, block, side and head.
struct ConvertUnit {
    char *codes, *wide;
    float* scale;
    int64_t token, wide_token;
    int rows;                 // token slots that hold tokens
};

__device__ __forceinline__ bool convert_unit(const ConvertArgs& a, int64_t u, ConvertUnit& unit) {
    const int head = int(u % a.kv_heads);
    int64_t rest = u / a.kv_heads;
    const int side = int(rest & 1);
    rest >>= 1;
    const int64_t i = rest % a.n;
    const int layer = int(rest / a.n);
    if (layer >= a.layers) return false;
    const kvsnap_c8_pair& p = a.pairs[layer];
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

template <typename T, int D>
__global__ void __launch_bounds__(256) compress_kernel(const __grid_constant__ ConvertArgs a) {
    constexpr int kLanes = D / 8, kRows = 32 / kLanes;
    const int lane = threadIdx.x % 32, sub = lane / kLanes, at = lane % kLanes * 8;
    ConvertUnit unit;
    if (!convert_unit(a, int64_t(blockIdx.x) * 8 + threadIdx.x / 32, unit)) return;
    float kept[kHeld][8], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int r = i * kRows + sub;
#pragma unroll
        for (int j = 0; j < 8; ++j) kept[i][j] = 0.0f;
        if (r < unit.rows) {
            load8<T>(unit.wide + r * unit.wide_token + 2 * at, kept[i]);
            amax = max8(kept[i], amax);
        }
    }
    for (int r = kHeld * kRows + sub; r < unit.rows; r += kRows) {
        float v[8];
        load8<T>(unit.wide + r * unit.wide_token + 2 * at, v);
        amax = max8(v, amax);
    }
    const float scale = needed_scale(warp_max(amax)), by = inverse(scale);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int r = i * kRows + sub;
        if (r < a.block_size) store_codes(unit.codes + r * unit.token + at, kept[i], by);
    }
    for (int r = kHeld * kRows + sub; r < a.block_size; r += kRows) {
        float v[8] = {};
        if (r < unit.rows) load8<T>(unit.wide + r * unit.wide_token + 2 * at, v);
        store_codes(unit.codes + r * unit.token + at, v, by);
    }
    if (lane == 0) *unit.scale = scale;
}

template <typename T, int D>
__global__ void __launch_bounds__(256) expand_kernel(const __grid_constant__ ConvertArgs a) {
    constexpr int kLanes = D / 8, kRows = 32 / kLanes;
    const int lane = threadIdx.x % 32, sub = lane / kLanes, at = lane % kLanes * 8;
    ConvertUnit unit;
    if (!convert_unit(a, int64_t(blockIdx.x) * 8 + threadIdx.x / 32, unit)) return;
    const float scale = *unit.scale;
    for (int r = sub; r < a.block_size; r += kRows) {
        float v[8];
        load_codes(unit.codes + r * unit.token + at, scale, v);
        store8<T>(unit.wide + r * unit.wide_token + 2 * at, v);
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
        check_batch(batch);
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
                           rotary_dim, query ? q_heads : 0, status};
        const bool single = batch->max_query <= 1;
        const int64_t units = single ? batch->seqs : batch->rows / cache->block_size + 2LL * batch->seqs;
        const dim3 grid(unsigned(units), unsigned((2 * cache->kv_heads + a.q_heads + 7) / 8));
        by_type(type, cache->head_dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int D = decltype(d)::value;
            const auto s = reinterpret_cast<cudaStream_t>(stream);
            if (single) {
                if (interleaved) append_kernel<T, D, true, true><<<grid, 256, 0, s>>>(a);
                else append_kernel<T, D, true, false><<<grid, 256, 0, s>>>(a);
            } else {
                if (interleaved) append_kernel<T, D, false, true><<<grid, 256, 0, s>>>(a);
                else append_kernel<T, D, false, false><<<grid, 256, 0, s>>>(a);
            }
        });
        check(cudaGetLastError());
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
        require(n < (1LL << 31) && 2 * n * layers / 8 * kv_heads < (1LL << 30), "too many blocks for one conversion");
        return true;
    }, [&] {
        const ConvertArgs a{pairs, ids, wide_ids, n, valid, layers, block_size, kv_heads, status};
        const int64_t ctas = (2 * n * layers * kv_heads + 7) / 8;
        by_type(type, head_dim, [&](auto t, auto d) {
            using T = decltype(t);
            constexpr int D = decltype(d)::value;
            const auto s = reinterpret_cast<cudaStream_t>(stream);
            if (EXPAND) expand_kernel<T, D><<<unsigned(ctas), 256, 0, s>>>(a);
            else compress_kernel<T, D><<<unsigned(ctas), 256, 0, s>>>(a);
        });
        check(cudaGetLastError());
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
