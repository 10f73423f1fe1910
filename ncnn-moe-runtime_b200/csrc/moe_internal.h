// Host-side declarations shared by the translation units of the library.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <mutex>
#include <new>
#include <string>
#include <vector>

#include "../../include/moe_b200_sampler.h"

#define MOE_SLICE_SLOT_RECORDS 1024u
// largest top_k the small-buffer kernel instantiation serves (the 4 * k + 64 records a slice expects above its sampled
// threshold must fit the 2048-record buffer with room for their spread)
#define MOE_SAMPLER_TOPK_SMALL_MAX 448u
// kept lists up to this length are verified in shared memory; longer ones need the dense residual scratch
#define MOE_SPECULATIVE_SHORT_LIST 1024u
// entries of the router's [expert][block] count table (expert_count * blocks of the select kernel never exceeds it)
#define MOE_ROUTER_BLOCK_TABLE_ENTRIES 262144u
// columns of an item of the quantisation, by its steps: the blocks of 128 that a half warp takes from it
#define MOE_QUANTIZE_ITEM 256u
// blocks of the balance loss's first kernel (its scratch holds one partial sum per block and expert): two per SM
#define MOE_BALANCE_MAX_BLOCKS 296u

namespace moe {

// Device workspace shared by the kernels of one handle.
struct Workspace
{
    // rows the streaming kernel could not finish; consumed (and reset to 0) by
    // the exact kernel of the same call
    uint32_t* exact_count = nullptr;   // [1]
    uint32_t* exact_done = nullptr;    // [1] CTAs of the exact kernel that have finished
    uint32_t* exact_next = nullptr;    // [1] next entry of exact_rows nobody has taken yet
    uint32_t* exact_rows = nullptr;    // [max_rows]
    // rows the clusters left to the one-CTA kernel of the same call (with a mark in the high bit), and their number
    uint32_t* exact_deferred = nullptr;       // [max_rows]
    uint32_t* exact_deferred_count = nullptr; // [1]
    // what the clusters did since it was last read, for tests (a row they leave has the same result): rows finished, rows
    // left, sums repeated with a corrected accumulator, sums repeated with better exponents
    uint32_t* cluster_counts = nullptr; // [4]
    uint32_t cluster_ctas = 0;          // CTAs per row; 0: chosen by the launcher
    // per-slot scratch of the exact kernels, stride = max_vocab rounded up to a multiple of 4 entries: two buffers of
    // 64-bit items for the one-CTA kernel; the cluster kernel before it keeps its items there (see ClusterSlice)
    uint32_t* sort_keys = nullptr;     // [slots][4][stride]
    // publication slots of the streaming kernel when a row is cut into slices:
    // one per CTA, MOE_SLICE_SLOT_RECORDS records and a 4-word header each
    uint64_t* slice_records = nullptr; // [slice_slots][MOE_SLICE_SLOT_RECORDS]
    uint32_t* slice_header = nullptr;  // [slice_slots][4]: count, needs-exact flag, max key, pad
    uint32_t* row_arrivals = nullptr;  // [max_rows] slices of the row that have published (self-resetting)
    uint32_t slice_slots = 0;
    uint32_t slots = 0;
    uint32_t max_rows = 0;
    uint32_t max_vocab = 0;
};

// The part [begin, end) of a row that one CTA of a cluster owns.  Slices begin at multiples of four logits and their items
// are written in whole groups of four, so a cluster's items end at the row's length rounded up to four: the numerators
// (4 B) fill at most the first of a slot's four arrays, the value groups (2 B) at most half of the second.
struct ClusterSlice
{
    uint32_t begin;
    uint32_t end;
};
__host__ __device__ inline ClusterSlice cluster_slice(uint32_t vocab, uint32_t cluster_size, uint32_t rank)
{
    const uint32_t per = ((vocab + cluster_size - 1u) / cluster_size + 3u) & ~3u;
    const uint64_t begin = static_cast<uint64_t>(rank) * per;
    if (begin >= vocab)
        return ClusterSlice{vocab, vocab}; // nothing left for it
    return ClusterSlice{static_cast<uint32_t>(begin), vocab - static_cast<uint32_t>(begin) < per ? vocab : static_cast<uint32_t>(begin) + per};
}

struct SampleArgs
{
    const void* logits;
    // a second logit matrix of the same stride that holds the rows from second_begin on (null: all rows are in `logits`)
    const void* logits_second;
    uint32_t second_begin;
    int dtype;
    uint32_t rows;
    uint32_t vocab;
    size_t row_stride;
    const moe_row_params* params; // device
    uint64_t step_offset;
    const int32_t* stop_offsets; // device or null
    const int32_t* stop_tokens;  // device or null
    int32_t* token_id;
    float* probability;
    uint32_t* row_flags;   // may be null
    int32_t* row_status;   // may be null
    // the four results above as one record per row instead (host-mapped memory of moe_sample_tokens); null: the arrays
    moe_sampled_row* packed;
    int32_t* topk_index;   // may be null
    uint32_t topk_stride;
    // optional: every row's kept candidates with their renormalised probabilities
    // (the vector sampling_distribution returns, session.cpp:76-136)
    int32_t* kept_token;     // [rows x kept_stride] or null
    float* kept_probability; // [rows x kept_stride] or null
    uint32_t* kept_count;    // [rows] or null: candidates kept (may exceed kept_stride; the list is cut there)
    uint32_t kept_stride;
    // vocabulary-sharded local pass: write the slice's Top-K records instead of sampling
    uint64_t* candidates_out; // may be null
    uint32_t candidates_k;
    uint32_t vocab_begin;
    // some row has a Top-K too large for the small record buffer: use the
    // large-buffer instantiation (fewer CTAs per SM)
    bool large_top_k;
    // moe_sampler_set_overlap: the streaming kernel reads its parameters and logits while the kernel before it is still
    // running and waits for that kernel (griddepcontrol.wait) before it touches anything else; without it the wait is
    // the first thing it does
    bool overlap_previous;
    // the exact kernels follow in the same call and may take their places on the SMs while this one runs
    bool release_exact;
};

cudaError_t launch_sample_rows(const SampleArgs& args, const Workspace& ws, uint32_t splits, cudaStream_t stream);
// untruncated_rows: how many rows of the batch have no Top-K (clusters take those; the other rows a batch may hand
// over have a Top-K above MOE_SAMPLER_TOPK_FAST_MAX)
cudaError_t launch_sample_exact(const SampleArgs& args, const Workspace& ws, uint32_t untruncated_rows, cudaStream_t stream);
cudaError_t launch_merge_candidates(const uint64_t* gathered, uint32_t shards, uint32_t rows, uint32_t top_k, const moe_row_params* params,
                                    uint64_t step_offset, int32_t* token_id, float* probability, uint32_t* row_flags, int32_t* row_status,
                                    int32_t* topk_index, uint32_t topk_stride, cudaStream_t stream);

// Speculative verification of `sessions` Sessions with draft_count proposals each.  Rows of the row
// outputs and kept lists: Session b's target positions are rows b*(draft_count+1) .. +draft_count,
// its draft positions rows sessions*(draft_count+1) + b*draft_count .. +draft_count-1.
struct SpeculativeArgs
{
    uint32_t sessions;
    uint32_t draft_count;
    uint32_t vocab;
    const moe_row_params* params; // device, by row; a Session's options and counters are those of its first target row
    const int32_t* proposed;      // device, [sessions * draft_count]
    const int32_t* token;         // per-row sampler outputs
    const float* probability;
    const uint32_t* row_flags;
    const int32_t* row_status;
    const int32_t* kept_token;
    const float* kept_probability;
    const uint32_t* kept_count;
    uint32_t kept_stride;
    float* dense;             // [sessions * vocab] scratch: the residual by token id
    int32_t* residual_token;  // [sessions * vocab] scratch: its positive entries in token-id order
    float* residual_value;
    float* accepted_probability; // [sessions * draft_count]
    moe_speculative_result* result; // [sessions]
};

cudaError_t launch_speculative_verify(const SpeculativeArgs& args, cudaStream_t stream);

struct RouterArgs
{
    const float* logits;
    uint32_t token_count;
    moe_router_options options; // pointers are device pointers
    uint32_t* expert_offsets;
    uint32_t* route_token;
    uint32_t* route_rank;
    float* route_weight;
    int32_t* plan_status;
    // scratch
    uint32_t* selected_expert; // [token_count * top_k]
    float* selected_weight;    // [token_count * top_k]
    uint32_t* block_counts;    // [MOE_ROUTER_BLOCK_TABLE_ENTRIES]: routes per (expert, block of the select kernel)
    uint32_t tokens_per_block; // filled in by the launcher
};
struct RouterPartition
{
    uint32_t tokens_per_block;
    uint32_t blocks;
};
// blocks of the select kernel: about four per SM (148 SMs, four warps of one token each per block), fewer when
// the [expert][block] table would outgrow MOE_ROUTER_BLOCK_TABLE_ENTRIES
inline RouterPartition router_partition_host(uint32_t token_count, uint32_t experts)
{
    constexpr uint32_t kWarpsPerBlock = 4;
    RouterPartition part;
    part.tokens_per_block = kWarpsPerBlock * ((token_count + kWarpsPerBlock * 592u - 1u) / (kWarpsPerBlock * 592u));
    if (part.tokens_per_block == 0)
        part.tokens_per_block = kWarpsPerBlock;
    part.blocks = (token_count + part.tokens_per_block - 1u) / part.tokens_per_block;
    while (static_cast<uint64_t>(part.blocks) * experts > MOE_ROUTER_BLOCK_TABLE_ENTRIES)
    {
        part.tokens_per_block *= 2u;
        part.blocks = (token_count + part.tokens_per_block - 1u) / part.tokens_per_block;
    }
    if (part.blocks == 0)
        part.blocks = 1;
    return part;
}
// expert_counts: [expert_count] scratch; scan_done: one word that is 0 between calls; error_word: ~0 between calls
cudaError_t launch_router_dispatch_kernels(const RouterArgs& args, uint32_t* expert_counts, uint32_t* scan_done, unsigned long long* error_word,
                                           cudaStream_t stream);
// out_of_range: one device word, set to 1 when a route_token entry is >= token_count (its row is zero-filled)
cudaError_t launch_regroup_gather(const float* hidden, uint32_t token_count, uint32_t columns, const uint32_t* route_token, uint32_t route_count,
                                  float* gathered, int32_t* out_of_range, cudaStream_t stream);

// Kernels that need more than 48 KiB of dynamic shared memory must opt in with
// cudaFuncSetAttribute, which applies to the current device only: what has been
// configured is remembered per device ordinal (one SharedOptIn per kernel).
constexpr int kMaxDevices = 64;
struct SharedOptIn
{
    std::mutex guard; // held from the look at `bytes` until the attribute is set: nobody launches in between
    size_t bytes[kMaxDevices] = {};
};
// true when `shared_bytes` still has to be configured on `device`; records it as configured (the caller holds the guard
// and configures it)
inline bool opt_in_needed(SharedOptIn& state, int device, size_t shared_bytes)
{
    if (device < 0 || device >= kMaxDevices)
        return true; // untracked ordinal: configure on every launch
    if (state.bytes[device] >= shared_bytes)
        return false;
    state.bytes[device] = shared_bytes;
    return true;
}
template<typename Kernel>
cudaError_t opt_in_shared(SharedOptIn& state, Kernel kernel, size_t shared_bytes)
{
    int device = 0;
    cudaError_t status = cudaGetDevice(&device);
    if (status != cudaSuccess)
        return status;
    const std::lock_guard<std::mutex> lock(state.guard);
    if (!opt_in_needed(state, device, shared_bytes))
        return cudaSuccess;
    status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared_bytes));
    if (status != cudaSuccess && device >= 0 && device < kMaxDevices)
        state.bytes[device] = 0;
    return status;
}

// Clusters of 1, 2, 4, 8 and 16 CTAs of one kernel that a device holds at once; 0: none of that size.
constexpr int kClusterSizes = 5;
struct ClusterOccupancy
{
    int active[kClusterSizes] = {};
};
struct ClusterOccupancyTable
{
    std::mutex guard;
    bool known[kMaxDevices] = {};
    ClusterOccupancy found[kMaxDevices];
};
// query(size_index, &clusters) -> cudaError_t.  Asked once per device, unless a size up to the portable 8 was not
// answered: then the call makes do with what it has (clusters of one CTA at least) and the next one asks again.
template<typename Query>
ClusterOccupancy cluster_occupancy(ClusterOccupancyTable& table, int device, Query query)
{
    const bool tracked = device >= 0 && device < kMaxDevices;
    const std::lock_guard<std::mutex> lock(table.guard);
    if (tracked && table.known[device])
        return table.found[device];
    ClusterOccupancy found;
    bool answered = true;
    for (int i = 0; i < kClusterSizes; ++i)
    {
        if (query(i, &found.active[i]) == cudaSuccess)
            continue;
        found.active[i] = 0;
        answered = answered && (1 << i) > 8;
    }
    if (found.active[0] < 1)
        found.active[0] = 1;
    if (tracked && answered)
    {
        table.found[device] = found;
        table.known[device] = true;
    }
    return found;
}

// A function that is looked up at run time: remembered once it is found.  A look-up that fails serves one call alone.
template<typename Function, typename LookUp>
Function found_once(std::atomic<Function>& found, LookUp look_up)
{
    Function function = found.load(std::memory_order_acquire);
    if (function == nullptr)
    {
        function = look_up();
        if (function != nullptr)
            found.store(function, std::memory_order_release);
    }
    return function;
}

// Scratch of calls that may be captured: what a captured graph was given stays allocated (in `kept`) until the handle goes, so
// a later, larger call does not take it away.  At least doubled each time where there is memory for that, so all of it together
// stays below twice the largest.  Nothing grows inside a capture: in the relaxed mode the allocation would succeed there, but a
// clearing would only be recorded, and a call before the first replay would find whatever the memory held.  pointer and capacity
// change only behind a clearing that was enqueued.
template<typename T>
cudaError_t grow_kept(std::vector<void*>& kept, T*& pointer, size_t& capacity, size_t wanted, cudaStream_t stream, bool cleared)
{
    if (wanted <= capacity)
        return cudaSuccess;
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    if (cudaError_t status = cudaStreamIsCapturing(stream, &capturing))
        return status;
    if (capturing != cudaStreamCaptureStatusNone)
        return cudaErrorStreamCaptureUnsupported;
    try
    {
        kept.reserve(kept.size() + 1u); // no exception may leave a C entry point
    }
    catch (const std::bad_alloc&)
    {
        return cudaErrorMemoryAllocation;
    }
    void* larger = nullptr;
    size_t entries = wanted > 2u * capacity ? wanted : 2u * capacity;
    cudaError_t status = cudaMalloc(&larger, entries * sizeof(T));
    if (status == cudaErrorMemoryAllocation && entries > wanted)
    {
        entries = wanted;
        status = cudaMalloc(&larger, entries * sizeof(T));
    }
    if (status != cudaSuccess)
    {
        (void)cudaGetLastError(); // it is reported here, not by the caller's next launch
        return status;
    }
    if (cleared)
    {
        status = cudaMemsetAsync(larger, 0, entries * sizeof(T), stream);
        if (status != cudaSuccess)
        {
            cudaFree(larger);
            return status;
        }
    }
    if (pointer != nullptr)
        kept.push_back(pointer);
    pointer = static_cast<T*>(larger);
    capacity = entries;
    return cudaSuccess;
}

// All kernels but the router's three launches (and the reset before them in moe_router_dispatch_static) are launched while
// the kernel before them in the stream may still run (programmatic stream serialization) and wait for it before they
// touch memory (wait_for_previous_kernel): the launch itself is out of the way when the earlier kernel ends.
// 1 to 3 us per launch.  The loads behind the wait are coherent ones: ld.global.nc and __ldg are for data that nobody
// writes while the kernel is resident.
inline cudaLaunchAttribute follow_closely()
{
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    return attribute;
}
template<typename... Parameters, typename... Arguments>
cudaError_t launch_following(void (*kernel)(Parameters...), uint32_t grid, uint32_t block, size_t shared_bytes, cudaStream_t stream, Arguments... arguments)
{
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid, 1, 1);
    config.blockDim = dim3(block, 1, 1);
    config.dynamicSmemBytes = shared_bytes;
    config.stream = stream;
    cudaLaunchAttribute attribute = follow_closely();
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<Parameters>(arguments)...);
}

// Stable Top-K of every row of `scores` (score descending, index ascending): out_index [rows x top_k] in that
// order, 0xFFFFFFFF beyond min(top_k, count); out_score may be null.  top_k <= MOE_INDEXER_TOPK_MAX.
cudaError_t launch_indexer_topk(const float* scores, uint32_t rows, uint32_t count, size_t row_stride, uint32_t top_k, uint32_t* out_index,
                                float* out_score, int sm_count, cudaStream_t stream);

// ---- expert products and balance ----

struct QuantizeArgs
{
    const void* source;
    uint32_t source_rows;
    uint32_t rows; // output rows
    uint32_t columns;
    size_t row_stride;
    const uint32_t* route_token; // [rows] or null
    uint8_t* values;
    float* scales;
    uint32_t* flags; // MOE_EXPERT_FLAG_* of the handle
};
struct ProductArgs
{
    const uint8_t* values;
    const float* scales;
    uint32_t rows;
    uint32_t columns;
    const uint8_t* weights;
    const float* weight_scales;
    uint32_t expert_count;
    uint32_t outputs;
    const uint32_t* expert_offsets; // null: all rows are expert 0's
    void* out;
    size_t out_stride;
    uint32_t* flags;
};
struct CombineArgs
{
    const void* route_rows;
    size_t row_stride;
    uint32_t columns;
    const uint32_t* route_token;
    const uint32_t* route_rank;
    const float* route_weight;
    uint32_t route_count;
    uint32_t token_count;
    uint32_t top_k;
    const void* base; // may be null
    void* out;
    uint32_t* slots; // [token_count * top_k], 0 between calls: route + 1 of every (token, rank)
    uint32_t* flags;
};
struct BalanceArgs
{
    const float* logits;
    uint32_t token_count;
    uint32_t expert_count;
    uint32_t top_k;
    int score_function;
    float coefficient;
    const uint8_t* token_mask; // may be null
    // forward only
    const uint32_t* expert_offsets;
    const uint32_t* route_token;
    uint32_t* expert_tokens;
    float* expert_probability;
    float* loss;
    float* partial_sums;      // [MOE_BALANCE_MAX_BLOCKS][expert_count]
    uint32_t* partial_counts; // [MOE_BALANCE_MAX_BLOCKS][expert_count + 1]
    float* partial_loss;      // [MOE_EXPERT_MAX_EXPERTS / 32]
    uint32_t* reduce_done;    // one word, 0 between calls
    uint32_t* flags;
};
// once: scratch of quantize_once_bytes for rows that are quantised once and then copied to their routes, or null
cudaError_t launch_quantize_rows(const QuantizeArgs& args, int dtype, int activation, uint8_t* once, cudaStream_t stream);
// Scratch for quantising each source row once, 0 where every route quantises its own row.  Dividing costs a value three times what
// copying a byte does, so large calls that use their rows often gain: 4096 rows x 4096 to 32768 routes 78 us route by route,
// 35 in two passes; 4096 rows x 2048 to 16384 routes 21.6 against 15.8.  To 8192 routes it costs (22 against 25 us), and so it does
// in small calls, by the second launch (1024 rows x 4096 to 4096 routes 11.6 against 16.2).  The quantised rows have to stay in L2
// between the passes, and are copied in 16-byte vectors.
constexpr size_t kQuantizeOnceBytes = 48u << 20; // the most, and what a handle allocates at its first such call
inline size_t quantize_once_bytes(const QuantizeArgs& a)
{
    const size_t values = (static_cast<size_t>(a.source_rows) * a.columns + 15u) / 16u * 16u;
    const size_t bytes = values + sizeof(float) * a.source_rows * ((static_cast<size_t>(a.columns) + MOE_EXPERT_BLOCK - 1u) / MOE_EXPERT_BLOCK);
    const bool worth = a.route_token != nullptr && a.rows / 4u >= a.source_rows && static_cast<uint64_t>(a.rows) * a.columns >= (1ull << 25);
    const bool fits = a.columns % 16u == 0u && reinterpret_cast<uintptr_t>(a.values) % 16u == 0u && a.source_rows > 0u && bytes <= kQuantizeOnceBytes;
    return worth && fits ? bytes : 0u;
}
// whether rows of source and values can be moved in vectors of eight values
inline bool quantize_in_vectors(const QuantizeArgs& a, size_t element)
{
    return a.columns % 8u == 0u && reinterpret_cast<uintptr_t>(a.source) % 16u == 0u && a.row_stride * element % 16u == 0u && reinterpret_cast<uintptr_t>(a.values) % 8u == 0u;
}
// Steps of a warp's item: four blocks a half warp share their divisions, in one pass over 1024 columns of a row, of which lanes stay
// empty where the row ends inside them; small calls wait for one item's latency.  So four steps are for calls of many values whose
// pieces of 256 columns fill those of 1024, to a share that hangs on what a value costs beside the divisions.  us with one and four
// steps, inputs from memory:
//   bf16        768 x 4096 4.1, 4.9; 1024 x 4096 5.5, 5.1; 2^25 values: x 256 31, 107; x 768 31, 40; x 1792 31, 32; x 2880 36, 28; x 5760 33, 29; x 4096 31, 24
//   bf16 gated  1024 x 4096 8.0, 8.3; 1300 x 4096 10.7, 10.0; 2^25: x 256 56, 164; x 768 56, 58; x 1280 57, 68; x 1792 57, 50; x 4096 57, 44
//   fp32        768 x 4096 4.4, 4.4; 1024 x 4096 5.4, 5.2; 2^25: x 256 28, 61; x 512 28, 34; x 1032 36, 33; x 2056 33, 29; x 4096 28, 27
//   fp32 gated  1536 x 4096 12.4, 14.1; 2048 x 4096 16.5, 17.1; 2^25: x 256 59, 217; x 2056 66, 83; x 2880 63, 62; x 4096 59, 58
//   rows that are not read in vectors: 1536 x 4095 bf16 11.8, 16.2, gated 15, 21; fp32 11.6, 13, gated 19, 20; 8194 x 4095 55, 54, 70, 74, 56, 54, 97, 89
inline uint32_t quantize_steps(const QuantizeArgs& a, size_t element, bool gate)
{
    const bool wide = element == 4u;
    const uint64_t most_small = gate && wide ? 16u << 20 : gate ? 4u << 20 : 3u << 20;                 // values
    const uint64_t filled = gate ? (wide ? 24u : 20u) : (wide ? 15u : 22u);                            // pieces of 256 for six of 1024
    const uint64_t pieces = (static_cast<uint64_t>(a.columns) + MOE_QUANTIZE_ITEM - 1u) / MOE_QUANTIZE_ITEM;
    const bool many = static_cast<uint64_t>(a.rows) * a.columns > (quantize_in_vectors(a, element) ? most_small : 16u << 20);
    return many && pieces * 6u >= (pieces + 3u) / 4u * filled ? 4u : 1u;
}
// whether a combine needs no slots: each of its CTAs looks through the routes
bool combine_few(uint32_t route_count, uint32_t token_count, uint32_t top_k);
cudaError_t launch_expert_product(const ProductArgs& args, int out_dtype, int sm_count, cudaStream_t stream);
cudaError_t launch_combine_routes(const CombineArgs& args, int dtype, cudaStream_t stream);
// Blocks of `warps` tokens each at a time, `most` of them at most.
inline uint32_t balance_blocks(uint32_t token_count, uint32_t warps, uint32_t most)
{
    const uint32_t wanted = token_count / warps + (token_count % warps != 0u ? 1u : 0u);
    return wanted < most ? wanted : most;
}
cudaError_t launch_balance_loss(const BalanceArgs& args, cudaStream_t stream);
cudaError_t launch_balance_loss_backward(const BalanceArgs& args, const uint32_t* expert_tokens, const float* loss_gradient, float* gradient, cudaStream_t stream);

// The checks of these calls that need no data: the text of the first one that fails, or null.
inline const char* check_value_type(int dtype)
{
    return dtype == MOE_DTYPE_F32 || dtype == MOE_DTYPE_BF16 ? nullptr : "dtype must be MOE_DTYPE_F32 or MOE_DTYPE_BF16";
}
inline bool misaligned(const void* pointer, size_t bytes)
{
    return reinterpret_cast<uintptr_t>(pointer) % bytes != 0u;
}
// value arrays of a caller's type start at a multiple of their element
inline bool misaligned_values(const void* pointer, int dtype)
{
    return misaligned(pointer, dtype == MOE_DTYPE_F32 ? 4u : 2u);
}
inline const char* check_quantize(const QuantizeArgs& a, int dtype, int activation)
{
    if (const char* text = check_value_type(dtype))
        return text;
    if (activation != MOE_ACTIVATION_NONE && activation != MOE_ACTIVATION_SILU_GATE)
        return "activation must be MOE_ACTIVATION_NONE or MOE_ACTIVATION_SILU_GATE";
    const size_t used = static_cast<size_t>(a.columns) * (activation == MOE_ACTIVATION_SILU_GATE ? 2u : 1u);
    if (a.row_stride < used)
        return "row_stride is smaller than the columns a row uses";
    if (a.columns > 0x7FFFFFFFu || a.rows > 0x7FFFFFFFu)
        return "columns and rows must be below 2^31";
    if (a.rows == 0 || a.columns == 0)
        return nullptr;
    if ((a.source == nullptr && a.source_rows > 0) || a.values == nullptr || a.scales == nullptr)
        return "source, values and scales must not be null";
    if (misaligned_values(a.source, dtype) || misaligned(a.scales, 4u) || misaligned(a.route_token, 4u))
        return "source, scales and route_token must be aligned to their elements";
    return nullptr;
}
inline const char* check_product(const ProductArgs& a, int out_dtype)
{
    if (check_value_type(out_dtype) != nullptr)
        return "out_dtype must be MOE_DTYPE_F32 or MOE_DTYPE_BF16";
    if (a.expert_count == 0 || a.expert_count > MOE_EXPERT_MAX_EXPERTS)
        return "expert products need 0 < expert_count <= MOE_EXPERT_MAX_EXPERTS";
    if (a.expert_offsets == nullptr && a.expert_count != 1)
        return "expert_offsets may only be null with one expert";
    if (a.columns == 0 || a.columns % 16u != 0)
        return "expert products need columns to be a positive multiple of 16";
    if (a.outputs == 0 || a.columns > 0x7FFFFFFFu || a.rows > 0x7FFFFFFFu || static_cast<uint64_t>(a.expert_count) * a.outputs > 0x7FFFFFFFull)
        return "expert products need outputs > 0 and rows, columns and expert_count * outputs below 2^31";
    if (a.out_stride < a.outputs)
        return "out_stride is smaller than outputs";
    if (a.rows == 0)
        return nullptr;
    if (a.values == nullptr || a.scales == nullptr || a.weights == nullptr || a.weight_scales == nullptr || a.out == nullptr)
        return "values, scales, weights, weight_scales and out must not be null";
    if (misaligned(a.values, 16u) || misaligned(a.weights, 16u))
        return "values and weights must be 16-byte aligned";
    if (misaligned(a.scales, 4u) || misaligned(a.weight_scales, 4u) || misaligned(a.expert_offsets, 4u) || misaligned_values(a.out, out_dtype))
        return "scales, weight_scales, expert_offsets and out must be aligned to their elements";
    return nullptr;
}
inline const char* check_combine(const CombineArgs& a, int dtype)
{
    if (const char* text = check_value_type(dtype))
        return text;
    if (a.row_stride < a.columns)
        return "row_stride is smaller than columns";
    if (a.columns > 0x7FFFFFFFu || a.token_count > 0x7FFFFFFFu || a.route_count > 0x7FFFFFFFu)
        return "columns, token_count and route_count must be below 2^31";
    if (a.token_count == 0 || a.columns == 0)
        return nullptr;
    if ((a.top_k == 0 && a.route_count > 0) || a.top_k > MOE_EXPERT_MAX_EXPERTS)
        return "combining needs 0 < top_k <= MOE_EXPERT_MAX_EXPERTS";
    if (a.out == nullptr)
        return "out must not be null";
    if (a.route_count > 0 && (a.route_rows == nullptr || a.route_token == nullptr || a.route_rank == nullptr || a.route_weight == nullptr))
        return "route_rows, route_token, route_rank and route_weight must not be null";
    if (misaligned_values(a.route_rows, dtype) || misaligned_values(a.base, dtype) || misaligned_values(a.out, dtype) || misaligned(a.route_token, 4u) ||
        misaligned(a.route_rank, 4u) || misaligned(a.route_weight, 4u))
        return "combine buffers must be aligned to their elements";
    return nullptr;
}
inline const char* check_balance(const BalanceArgs& a)
{
    if (a.score_function != MOE_ROUTER_SOFTMAX && a.score_function != MOE_ROUTER_SIGMOID && a.score_function != MOE_ROUTER_SQRT_SOFTPLUS)
        return "score_function must be a moe_router_score";
    if (!(a.coefficient - a.coefficient == 0.0f))
        return "the balance coefficient must be finite";
    if (misaligned(a.logits, 4u) || misaligned(a.expert_offsets, 4u) || misaligned(a.route_token, 4u) || misaligned(a.expert_tokens, 4u) ||
        misaligned(a.expert_probability, 4u) || misaligned(a.loss, 4u))
        return "balance buffers must be aligned to their elements";
    return nullptr;
}

uint32_t choose_splits(uint32_t rows, uint32_t vocab, int dtype, int sm_count, uint32_t slice_slots, bool large_top_k, bool overlapped);

} // namespace moe

// ---- for tests; not part of the ABI ----
// Fixes the CTAs per row of the handle's clusters (1, 2, 4, 8 or 16; 0: chosen by the launcher).
extern "C" int moe_internal_set_cluster_ctas(moe_sampler* sampler, uint32_t ctas);
// Synchronises `stream`, copies Workspace::cluster_counts to the host and clears them.
extern "C" int moe_internal_cluster_counts(moe_sampler* sampler, void* stream, uint32_t* counts);
