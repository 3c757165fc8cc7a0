/*
 * kvsnap_cuda.h: the C ABI of kvsnap_b200/_native/_cuda_native.so.
 *
 * Three groups of entry points, all extern "C", plain pointers and sizes, no
 * torch types. Every int-returning call returns 0 on success and -1 on error,
 * with the message in the calling thread's kvsnap_cuda_error().
 *
 * 1. The pinned-pool ABI, version 2: the same symbols, argument meaning and
 *    error behaviour as the reference's csrc/dataplane/cuda_pool.cpp, which
 *    kvsnap/connector/dataplane.py:47-60 binds with ctypes. A build of this
 *    library dropped in as kvsnap/_native/_cuda_native<EXT_SUFFIX>.so (or named
 *    by KVSNAP_CUDA_LIBRARY) serves the reference's CudaPool unchanged.
 *
 * 2. The data-plane kernels (kvsnap_dp_*), sm_100a CUDA. They replace the
 *    reference's restore kernel (kvsnap/connector/copy_kernel.py:23-49), its
 *    torch save gather (kvsnap/connector/dataplane.py:409-427) and its host
 *    checksums (csrc/dataplane/io.cpp:27-47 CRC32C, hashlib SHA-256 in
 *    kvsnap/store/store.py:616-629 and kvsnap/connector/volatile.py:141-151).
 *    Tables passed to them (spans, block ids, addresses) live in device memory
 *    (or mapped pinned memory); packed-block addresses may be device memory or
 *    pinned host memory from cudaHostAlloc, which the kernels read and write in
 *    place over the host link.
 *
 * 3. The 8-bit paged KV cache (kvsnap_c8_*): appending to it, attention over
 *    it, and conversion of blocks between it and a 16-bit cache.
 */
#ifndef KVSNAP_CUDA_H
#define KVSNAP_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- 1. pinned pool (ABI 2) ------------------------------------------------ */

/* Thread-local text of the last error (reference cuda_pool.cpp:50). */
const char* kvsnap_cuda_error(void);
/* Returns 2 (reference cuda_pool.cpp:52; checked at dataplane.py:64-66). */
int kvsnap_pool_abi_version(void);
/* A pinned arena of `capacity` bytes on `device` plus its own non-blocking copy
   stream; NULL on error (reference cuda_pool.cpp:53-62). */
void* kvsnap_pool_create(size_t capacity, int device);
/* Frees the pool; if its stream cannot be drained the pinned memory is kept
   (quarantined) instead of freed (reference cuda_pool.cpp:63, 30-38). */
void kvsnap_pool_destroy(void* pool);
/* Drains the copy stream, then frees; on a failed drain the pool stays intact
   and -1 is returned (reference cuda_pool.cpp:66-74). */
int kvsnap_pool_close_checked(void* pool);
/* The copy stream's handle, borrowed (reference cuda_pool.cpp:78-85). */
int kvsnap_pool_copy_stream(void* pool, uintptr_t* stream);
/* First-fit reservation. Fails with a message containing "pinned capacity
   exhausted" when it cannot fit (reference cuda_pool.cpp:86-104). Start offsets
   are rounded up to 16 bytes so every allocation suits 16-byte vector access. */
int kvsnap_pool_reserve(void* pool, size_t size, uint64_t* id, void** ptr);
/* One async copy between device memory and an allocation on the copy stream;
   a device-to-host copy first waits for `producer_stream` (reference
   cuda_pool.cpp:107-133). */
int kvsnap_pool_copy(void* pool, uint64_t id, size_t host_offset, void* device_ptr, size_t size, int to_host,
                     uintptr_t producer_stream);
/* `height` rows of `width` bytes, strided on both sides (reference cuda_pool.cpp:139-169). */
int kvsnap_pool_copy_2d(void* pool, uint64_t id, size_t host_offset, size_t host_pitch, void* device_ptr,
                        size_t device_pitch, size_t width, size_t height, int to_host, uintptr_t producer_stream);
/* Block until the allocation's last copy completes (reference cuda_pool.cpp:170-177). */
int kvsnap_pool_wait(void* pool, uint64_t id);
/* 1 when idle, 0 while a copy is in flight, -1 on error (reference cuda_pool.cpp:178-189). */
int kvsnap_pool_ready(void* pool, uint64_t id);
/* Wait, then return the bytes to the arena (reference cuda_pool.cpp:190-199). */
int kvsnap_pool_release(void* pool, uint64_t id);
/* Extension (no reference counterpart): kvsnap_pool_copy queued on `stream`
   (0: the pool's copy stream) instead of the pool's stream, with no producer
   fence: the caller orders its own stream. Lets a restore's host-to-device
   copies run beside a save's device-to-host copies (the host link is full
   duplex). The allocation's completion event is recorded on `stream`. */
int kvsnap_pool_copy_on(void* pool, uint64_t id, size_t host_offset, void* device_ptr, size_t size, int to_host,
                        uintptr_t stream);
/* Extension (no reference counterpart): record the allocation's completion
   event on `stream` (0: the pool's copy stream) now, so wait/ready/release
   also fence kernels queued there that read or write the allocation in place. */
int kvsnap_pool_mark(void* pool, uint64_t id, uintptr_t stream);
/* Extension (no reference counterpart): n copies in one call, entry k moving
   sizes[k] bytes between allocation ids[k] at host_offsets[k] and device
   address device_ptrs[k], queued in order on `stream` (0: the pool's copy
   stream) with no producer fence. Every entry is checked before any is
   queued; each allocation's completion event is recorded after the last copy.
   Consecutive entries whose host and device ranges both continue the previous
   one's move in one copy.
   Replaces n kvsnap_pool_copy_on calls (one per block of a host-tier
   snapshot, reference volatile.py:281-307) with one. */
int kvsnap_pool_copy_many(void* pool, int64_t n, const uint64_t* ids, const uint64_t* host_offsets,
                          const uint64_t* device_ptrs, const uint64_t* sizes, int to_host, uintptr_t stream);
/* Extension: kvsnap_pool_wait for each of n allocations, in one call. */
int kvsnap_pool_wait_many(void* pool, int64_t n, const uint64_t* ids);

/* Extension for the cross-owner host tier (replaces the socket copy of
   kvsnap/connector/vllm.py:524-534 and connector/volatile.py:87-138): a pool
   whose arena is POSIX shared memory named `name` (one path component that
   starts with '/', created with mode 0600, so only this user's processes open
   it), registered with CUDA as pinned and mapped memory. It behaves as
   kvsnap_pool_create's; destroying it unlinks the name, and the mappings other
   processes made stay valid until they close them. NULL on error (a name
   already in use included). */
void* kvsnap_pool_create_shared(size_t capacity, int device, const char* name);
/* Extension: the arena's first byte and its capacity, so an owner can tell
   other processes where an allocation lies in its shared arena. */
int kvsnap_pool_arena(void* pool, void** base, size_t* capacity);
/* Map another process's shared arena read-only into this one and register it
   with CUDA (pinned, mapped, read-only) on `device`, so that its blocks serve
   as restore sources in place: *base and *size receive the mapping. */
int kvsnap_shared_open(const char* name, int device, void** base, size_t* size);
/* Unregister and unmap a mapping from kvsnap_shared_open. The caller first
   waits for every copy and kernel that reads it. */
int kvsnap_shared_close(void* base, size_t size);

/* ---- 2. data-plane kernels --------------------------------------------------- */

#define KVSNAP_DP_ABI_VERSION 1

/* Status bits a kernel ORs into its status word instead of faulting. */
#define KVSNAP_DP_MISALIGNED 1u      /* an address or size broke the vector width */
#define KVSNAP_DP_BAD_BLOCK 2u       /* a block id outside its cache */
#define KVSNAP_DP_CRC_MISMATCH 4u    /* a block's CRC32C differed from the expected one */
#define KVSNAP_DP_BAD_CUT 8u         /* KVSNAP_DP_PAIRS or _SPLIT* met spans that do not cut that way */

/* OR into a `vec` argument when every packed address is device memory: the
   kernels then cut each unit into 4 segments, move whole 128-byte lines
   coalesced, each group of 8 lanes 1 KiB of its segment a step, and CRC each
   lane's bytes in its registers through per-lane tables (HBM-friendly),
   instead of 16 bytes a lane in 512-byte steps (host-link friendly).
   Needs vec 16. */
#define KVSNAP_DP_HBM 0x100
/* With KVSNAP_DP_HBM, a hint when every span is small (up to 8 KiB, e.g. a
   tensor-parallel shard's): each warp then takes contiguous units and folds
   the CRCs of a block's consecutive spans as one run. Results are the same
   with or without it. */
#define KVSNAP_DP_RUNS 0x200
/* With KVSNAP_DP_RUNS, a hint when every span has one size S of 2 or 4 KiB
   (a TP-8 or TP-16 shard's) and nspans is even: each unit is then a pair of
   consecutive spans, so each lane owns 2 * S / 32 contiguous packed bytes and
   a unit's CRC is placed once per 2 * S. A pair whose spans differ sets
   KVSNAP_DP_BAD_CUT and is skipped. Results are the same with or without
   it. */
#define KVSNAP_DP_PAIRS 0x400
/* With KVSNAP_DP_HBM, without KVSNAP_DP_RUNS: each unit is one of 2 (SPLIT2)
   or 4 (SPLIT4) equal pieces of a span, so that large spans (a Qwen3-8B
   layer's 32 KiB) move in 16 KiB units, which measured faster. Every span
   must cut into pieces that are a multiple of 4 KiB; one that does not sets
   KVSNAP_DP_BAD_CUT and is skipped. The last block of a gather with
   valid_tokens > 0 is not split. Results are the same with or without it. */
#define KVSNAP_DP_SPLIT2 0x800
#define KVSNAP_DP_SPLIT4 0x1000
#define KVSNAP_DP_SPLIT_MASK 0x1800
/* With KVSNAP_DP_HBM and crc_out: add this call's share of each block's CRC
   to crc_out as it stands (not cleared first) and leave it raw (no finish
   step). A save that moves each block in several calls, a range of spans at
   a time, ends with kvsnap_dp_crc32c_finish. */
#define KVSNAP_DP_CRC_ACCUMULATE 0x2000

/*
 * One registered layer view, i.e. one span of every packed block. A packed
 * block is the spans back to back in registration order (layer-name order,
 * reference dataplane.py:226); span s of cache block b lives at
 * base + b * pitch and is `bytes` long, dense, copied in storage order
 * (dataplane.py:283-305). 64 bytes.
 */
typedef struct kvsnap_span {
    int64_t base;         /* device address of block 0 of this view */
    int64_t pitch;        /* bytes between consecutive blocks */
    int64_t offset;       /* byte offset of the span inside a packed block */
    int64_t bytes;        /* span bytes per block */
    int64_t token_pitch;  /* bytes between consecutive token slots (tail zeroing) */
    int32_t tokens;       /* token slots per block (the block size) */
    int32_t row_bytes;    /* contiguous bytes of one (head, token) row */
    int64_t nblocks;      /* blocks in this cache, for in-kernel bounds checks */
    uint32_t crc_shift;   /* x^(8 * bytes after this span) mod P, filled by kvsnap_dp_plan */
    uint32_t flags;       /* reserved, 0 */
} kvsnap_span;

int kvsnap_dp_abi_version(void);

/* Fill `offset` and `crc_shift` of a host span array in registration order;
   writes the packed block size to *block_bytes. Host-only, no CUDA. */
int kvsnap_dp_plan(kvsnap_span* spans, int nspans, uint64_t* block_bytes);

/* CRC32C of a host buffer with a prior value: the host library's semantics
   (reference io.cpp:39-44), exported here for self-checks. Host-only. */
uint32_t kvsnap_dp_crc32c_host(const void* data, size_t size, uint32_t prior);

/*
 * Save gather (replaces dataplane.py:388-437 and its host hashing). For each
 * i < n and span s: copy the span of cache block blocks[i] to
 * targets[i] + spans[s].offset. In block n-1, token slots >= valid_tokens are
 * written as zeros when valid_tokens > 0 (dataplane.py:262-272, 433-436).
 * When crc_out is not NULL, crc_out[i] receives the CRC32C of packed block i
 * as written (zeros included). `vec` is 16 or 8: the alignment every address,
 * pitch, offset and span size meets. `ctas` 0 picks a default. status (device
 * word, may be NULL) receives KVSNAP_DP_* bits.
 */
int kvsnap_dp_gather(const kvsnap_span* spans, int nspans, uint64_t block_bytes, const int64_t* blocks,
                     const int64_t* targets, int64_t n, int32_t valid_tokens, uint32_t* crc_out,
                     uint32_t* status, int vec, int ctas, uintptr_t stream);

/*
 * Restore scatter (replaces copy_kernel.py:23-49 and the loader-thread CRC
 * check, store.py:717-718). For each i < n and span s: copy
 * sources[i] + spans[s].offset to the span of cache block blocks[i]. When
 * crc_out is not NULL it receives the CRC32C of each source block; when
 * expect is not NULL as well, a block whose CRC differs sets
 * KVSNAP_DP_CRC_MISMATCH in *status (its bytes are already written: callers
 * that must not write unverified bytes verify first with kvsnap_dp_crc32c).
 * A non-NULL `gate` is read by every CTA first: when *gate is non-zero the
 * kernel writes nothing.
 */
int kvsnap_dp_scatter(const kvsnap_span* spans, int nspans, uint64_t block_bytes, const int64_t* sources,
                      const int64_t* blocks, int64_t n, uint32_t* crc_out, const uint32_t* expect,
                      const uint32_t* gate, uint32_t* status, int vec, int ctas, uintptr_t stream);

/* CRC32C of n packed blocks of block_bytes at addrs[i] (device or pinned host).
   With expect not NULL, mismatches set KVSNAP_DP_CRC_MISMATCH in *status. */
int kvsnap_dp_crc32c(const int64_t* addrs, int64_t n, uint64_t block_bytes, uint32_t* crc_out,
                     const uint32_t* expect, uint32_t* status, int vec, int ctas, uintptr_t stream);

/* SHA-256 of n packed blocks of block_bytes at addrs[i]; digest i is the 32
   big-endian bytes at out + 32 * i, the bytes of hashlib.sha256(block).digest()
   (the store's content id, store.py:623). One lane hashes one block. */
int kvsnap_dp_sha256(const int64_t* addrs, int64_t n, uint64_t block_bytes, uint8_t* out, uintptr_t stream);

/* The same hash, one part of every block at a time, so that the bytes of only
   one part need to be in device memory at once. Call it for parts in order:
   bytes [done_bytes, done_bytes + part_bytes) of each block of total_bytes,
   that part starting at addrs[i]. state holds 8 words a block between calls
   (n * 32 bytes, device memory): the first part (done_bytes 0) starts from
   the SHA-256 initial value, later ones from state. Parts before the last
   must be whole 64-byte chunks; the last part (done_bytes + part_bytes ==
   total_bytes) pads and writes the digests to out as kvsnap_dp_sha256 does,
   the others write state. */
int kvsnap_dp_sha256_part(const int64_t* addrs, int64_t n, uint64_t part_bytes, uint64_t done_bytes,
                          uint64_t total_bytes, uint32_t* state, uint8_t* out, uintptr_t stream);

/* Land one column of n packed blocks from a device slot where each block goes:
   bytes [0, len) at src + i * src_stride are copied to targets[i] + offset,
   for i < n. Targets may be pinned host memory (written over the host link by
   the SMs, one 4 KiB piece a warp step) or device memory. No counterpart in
   the reference: its save copies whole chunks with cudaMemcpyAsync
   (kvsnap/connector/dataplane.py:418-427); a bounded save's columns are too
   small for the copy engine (256 KiB copies to scattered per-block targets ran
   at 30 GB/s on B200, this kernel at 52.6 with 16 CTAs). src, src_stride,
   offset, len and every target must be multiples of 16 bytes: a block that
   is not sets KVSNAP_DP_MISALIGNED in *status and is skipped. `ctas` 0 picks 16. */
int kvsnap_dp_land(const void* src, int64_t src_stride, const int64_t* targets, int64_t offset, int64_t n,
                   int64_t len, uint32_t* status, int ctas, uintptr_t stream);

/* Land one column of n packed blocks whose targets lie at one pitch: bytes
   [0, len) at src + i * src_stride are copied to dst + i * dst_pitch, for
   i < n, as one copy-engine transfer (cudaMemcpy2DAsync, device to host) on
   `stream`. dst is pinned host memory. A bounded save's column is n small
   pieces, so when its targets are evenly spaced (blocks reserved back to back,
   or one buffer) this moves the column at the copy engine's rate while the SMs
   gather the next one; otherwise kvsnap_dp_land. No counterpart in the
   reference, whose save copies whole chunks with cudaMemcpyAsync
   (kvsnap/connector/dataplane.py:418-427). */
int kvsnap_dp_land_strided(const void* src, int64_t src_stride, void* dst, int64_t dst_pitch, int64_t n,
                           int64_t len, uintptr_t stream);

/* Finish raw CRC accumulators that KVSNAP_DP_HBM gathers or scatters left
   under KVSNAP_DP_CRC_ACCUMULATE: crc[i] becomes block i's CRC32C; with
   expect not NULL, mismatches set KVSNAP_DP_CRC_MISMATCH in *status. */
int kvsnap_dp_crc32c_finish(uint32_t* crc, const uint32_t* expect, int64_t n, uint64_t block_bytes,
                            uint32_t* status, uintptr_t stream);

/*
 * The reference restore kernel's exact interface (copy_kernel.py:43-49): all
 * six tables are device int64 arrays; job j copies layer_words[l] 8-byte words
 * of layer l = j % n_layers from sources[b] + layer_offsets[l] to
 * layer_bases[l] + blocks[b] * layer_pitches[l], b = j / n_layers. No checksums.
 */
int kvsnap_dp_copy_host_blocks(const int64_t* sources, const int64_t* blocks, int64_t n_blocks,
                               const int64_t* layer_offsets, const int64_t* layer_bases,
                               const int64_t* layer_pitches, const int64_t* layer_words, int64_t n_layers,
                               int ctas, uintptr_t stream);

/*
 * Tensor-parallel regroup (no reference counterpart: the reference treats a
 * restore at another TP size as a miss, kvsnap/connector/vllm.py:9-14). This
 * rank's cache holds H heads a layer; the snapshot was saved by `groups` times
 * as many ranks, shard q holding heads [q*H/groups, (q+1)*H/groups). For each
 * block i and span s, every (head, token) row of cache block blocks[i] is read
 * from shard q's packed block at shards[i*groups + q] + src_spans[s].offset.
 * src_spans describe one shard's packed layout (the same spans with H/groups
 * heads; offsets from kvsnap_dp_plan). Shard addresses may be this GPU's
 * memory or a peer's mapped with kvsnap_dp_ipc_open: the kernel reads them
 * with plain loads over NVLink. The caller orders producer and consumer ranks.
 */
int kvsnap_dp_regroup(const kvsnap_span* dst_spans, const kvsnap_span* src_spans, int nspans, const int64_t* shards,
                      int groups, const int64_t* blocks, int64_t n, uint32_t* status, int ctas, uintptr_t stream);

/* Device memory from cudaMalloc, shareable with other processes through
   kvsnap_dp_ipc_export (memory from torch's expandable segments is not). */
int kvsnap_dp_device_alloc(size_t size, int device, void** ptr);
int kvsnap_dp_device_free(void* ptr);
/* A 64-byte CUDA IPC handle for an allocation made by kvsnap_dp_device_alloc. */
int kvsnap_dp_ipc_export(void* ptr, void* handle);
/* Map another process's allocation into this one on `device` (peer access enabled lazily). */
int kvsnap_dp_ipc_open(const void* handle, int device, void** ptr);
int kvsnap_dp_ipc_close(void* ptr);

/*
 * Verified restore scatter that allocates nothing. No counterpart in the
 * reference. For callers that cannot allocate device memory: a serving worker
 * whose KV cache was sized to fill the GPU has no room left for a CRC buffer,
 * and host code that must not enter an allocator (which may synchronise the
 * device) cannot ask for one. The per-block CRC32C accumulators and one gate
 * word live in one fixed scratch array inside this library,
 * (KVSNAP_DP_STATIC_MAX_BLOCKS + 64) x 4 bytes, held on every GPU that loads
 * the library until the process exits. The caller passes inputs and outputs.
 *
 * Check before write: every source block's CRC32C is computed and compared
 * with expect[i] first; the scatter then runs gated on that verdict. On a
 * mismatch nothing is written to the cache and KVSNAP_DP_CRC_MISMATCH is set
 * in *status (other bits as kvsnap_dp_scatter sets them). `vec` takes the same
 * flags as kvsnap_dp_scatter (KVSNAP_DP_HBM and its unit cuts for sources in
 * device memory). Sources in pinned host memory cross the host link twice,
 * once for the check and once for the copy.
 *
 * n above the maximum is rejected with an error and nothing is launched.
 * Every call looks up the scratch's device address (cudaGetSymbolAddress, no
 * allocation); make the first call on a device before any stream capture,
 * since it may load the module. Every call shares the scratch and clears what
 * it uses at its start: calls whose work overlaps on the GPU race on it and
 * must not be issued concurrently.
 */
#define KVSNAP_DP_STATIC_MAX_BLOCKS 65536
int kvsnap_dp_scatter_verify_static(const kvsnap_span* spans, int nspans, uint64_t block_bytes,
                                    const int64_t* sources, const int64_t* blocks, int64_t n,
                                    const uint32_t* expect, uint32_t* status, int vec, int ctas, uintptr_t stream);

/* ---- 3. the 8-bit paged KV cache ------------------------------------------------ */

/*
 * A layer's paged cache in 8 bits: e4m3 codes [2 sides, blocks, block_size,
 * kv_heads, head_dim] (side 0 keys, 1 values; last axis contiguous, the other
 * pitches in bytes and multiples of 16, as the base), and one float scale a
 * block, side and KV head, scales[block][side][head], contiguous. A code c at
 * scale s stands for c * s. Scales written here are powers of two: the
 * smallest s >= 2^-126 with largest finite magnitude <= 448 s, and 0 for a
 * block of zeros. No counterpart in the reference, which moves caches and
 * never reads one.
 */
typedef struct kvsnap_c8_cache {
    int64_t codes;            /* device address of block 0's first key code */
    int64_t scales;           /* device address of scales[0][0][0] */
    int64_t side_pitch, block_pitch, token_pitch, head_pitch;
    int32_t blocks, block_size, kv_heads, head_dim;
    int32_t device, reserved;
} kvsnap_c8_cache;

/*
 * The sequences of one call. Sequence s owns the token rows start[s] ..
 * start[s+1]-1 of the call's tensors; they are its last tokens, lengths[s]
 * tokens long with them. Its token at position p lies in block
 * table[s * table_pitch + p / block_size], slot p % block_size. Rows from
 * start[seqs] on belong to nobody. A row whose position would be negative
 * (lengths[s] below the row count, 0 for a padded entry) is not in the cache.
 * All three arrays are device memory, read by the kernels, never by the host.
 * A table row holds at most 2^30 tokens.
 */
typedef struct kvsnap_c8_batch {
    int64_t table, start, lengths;      /* device addresses of int32 arrays */
    int64_t table_pitch;                /* elements between the table's rows */
    int32_t width;                      /* blocks a row of the table holds */
    int32_t seqs, rows;                 /* sequences; token rows of the call's tensors */
    int32_t max_query;                  /* no sequence has more rows than this */
} kvsnap_c8_batch;

/* 16-bit element types. */
#define KVSNAP_C8_BF16 0
#define KVSNAP_C8_FP16 1

/* Status bits beside KVSNAP_DP_BAD_BLOCK (a table entry outside the cache). A
   kernel that sets one has skipped what the bit is about, not faulted. */
#define KVSNAP_C8_BAD_LENGTH 16u     /* lengths, start or max_query do not fit the table or the rows */
#define KVSNAP_C8_BAD_POSITION 32u   /* a position behind the rotary table's end: its token is left out */
#define KVSNAP_C8_STALLED 64u        /* a wait inside a kernel ran out (two seconds): its results are not valid */

/*
 * Append: key and value rows [rows][kv_heads][head_dim] (token and head
 * pitches in bytes, multiples of 16) into their pages. With rotary not NULL,
 * keys are first rotated in 32 bits: rotary[p][i] = (cos, sin) of the angle of
 * pair i at position p, i < rotary_dim / 2, floats; pair i is elements (i, i +
 * rotary_dim / 2), or (2i, 2i + 1) with interleaved; elements from rotary_dim
 * on pass unchanged. One rounding, to the code. With query not NULL its rows
 * are rotated the same way into query_out, dense [rows][q_heads][head_dim].
 * A page that already holds tokens of its sequence keeps its scale or grows it
 * to what the new tokens need, and its older codes are then rounded again at
 * the new scale; a page whose first slot is written starts anew. Slots behind
 * the last token keep their codes. Tokens behind the rotary table's last
 * position, and all of a sequence that does not fit, are left out. Infinities become the largest value the
 * block's scale holds, NaN stays NaN. Two sequences that append in one call
 * must not share the page they append to.
 */
int kvsnap_c8_append(const kvsnap_c8_cache* cache, const kvsnap_c8_batch* batch, int type, const void* key,
                     int64_t key_token, int64_t key_head, const void* value, int64_t value_token,
                     int64_t value_head, const void* query, int64_t query_token, int64_t query_head, int q_heads,
                     void* query_out, const float* rotary, int64_t positions, int rotary_dim, int interleaved,
                     uint32_t* status, uintptr_t stream);

/*
 * Attention of query rows [rows][q_heads][head_dim] over their sequences'
 * cached tokens: out[i][h] = sum_j softmax_j(scale * q.k_j) v_j over positions j
 * up to the row's own. Query heads g * q_heads / kv_heads .. share KV head g.
 * A row that sees no token is zeros; rows that belong to nobody, or to a
 * sequence that does not fit, are not written. out may be query if that is
 * dense. A weight times its page's value scale is rounded to 16 bits once,
 * relative to the row's largest such product. out is dense and of the query's type. The workspace is device memory,
 * 16-byte aligned, of at least kvsnap_c8_attend_workspace's bytes for the same
 * cache, batch and heads; calls that may overlap need one each. What it holds
 * before does not matter.
 */
int kvsnap_c8_attend(const kvsnap_c8_cache* cache, const kvsnap_c8_batch* batch, int type, const void* query,
                     int64_t query_token, int64_t query_head, int q_heads, float scale, void* out, void* workspace,
                     size_t workspace_bytes, uint32_t* status, uintptr_t stream);
int kvsnap_c8_attend_workspace(const kvsnap_c8_cache* cache, const kvsnap_c8_batch* batch, int q_heads,
                               size_t* bytes);

/* One layer of a conversion: the 8-bit cache and a 16-bit one of the same
   block_size, kv_heads and head_dim (pitches as in kvsnap_c8_cache). */
typedef struct kvsnap_c8_pair {
    int64_t codes, scales, side_pitch, block_pitch, token_pitch, head_pitch;
    int64_t wide, wide_side, wide_block, wide_token, wide_head;
    int32_t blocks, wide_blocks;
} kvsnap_c8_pair;

/*
 * Whole blocks between a 16-bit cache and the 8-bit one, every layer in one
 * launch: pairs is a device array of `layers`, wide_ids and ids device int64
 * arrays of n block ids. compress writes blocks ids[i] from wide_ids[i]; token
 * slots from valid_tokens on (counted over the n blocks; negative: none) become
 * zeros. expand writes blocks wide_ids[i] from ids[i], rounded once. No block
 * may be written twice in one call.
 */
int kvsnap_c8_compress(const kvsnap_c8_pair* pairs, int layers, int block_size, int kv_heads, int head_dim, int type,
                       const int64_t* wide_ids, const int64_t* ids, int64_t n, int64_t valid_tokens,
                       uint32_t* status, int device, uintptr_t stream);
int kvsnap_c8_expand(const kvsnap_c8_pair* pairs, int layers, int block_size, int kv_heads, int head_dim, int type,
                     const int64_t* ids, const int64_t* wide_ids, int64_t n, uint32_t* status, int device,
                     uintptr_t stream);

#ifdef __cplusplus
}
#endif
#endif /* KVSNAP_CUDA_H */
