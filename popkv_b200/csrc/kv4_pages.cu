// Pages of the 4-bit cache: share, extend (with copy on write), truncate, copy
// and compact, all from device-resident tables, so that a captured graph or a
// serving loop needs no host round trip.
//
// A page is free exactly when its reference count is 0; new pages are the lowest
// free ones, so the result depends on the tables alone.
//
// The plans are one CTA each and bound by latency (fork, extend: a chain of four to six
// dependent loads and block scans, 4 to 6 us); the copies by memory: compacting 0.54 GB in
// 32 layers takes 196 us, 164 at the copy rate.  A fork into 8 branches that each write a
// token, copies of 21 MB among it, takes 16.5 us.
#include "kv4.cuh"

namespace popkv {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kRowThreads = 128;
constexpr int kMostEntries = 4096;  // sequences of one call

// Whether entry i names a sequence in range that no earlier entry names.
__device__ bool first_of(const Kv4View& view, const int32_t* seqs, int i) {
    const int s = seqs[i];
    if (!view.has_sequence(s)) return false;
    for (int j = 0; j < i; ++j)
        if (seqs[j] == s) return false;
    return true;
}

// Exclusive prefix sum over the block (kPlanThreads threads); *total for everybody.
template <typename T>
__device__ T block_scan(T value, T* total) {
    __shared__ T sums[kPlanThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T inclusive = value;
#pragma unroll
    for (int step = 1; step < 32; step *= 2) {
        const T other = __shfl_up_sync(0xFFFFFFFFu, inclusive, step);
        if (lane >= step) inclusive += other;
    }
    if (lane == 31) sums[warp] = inclusive;
    __syncthreads();
    if (warp == 0) {
        T s = sums[lane];
#pragma unroll
        for (int step = 1; step < 32; step *= 2) {
            const T other = __shfl_up_sync(0xFFFFFFFFu, s, step);
            if (lane >= step) s += other;
        }
        sums[lane] = s;
    }
    __syncthreads();
    const T before = warp ? sums[warp - 1] : 0;
    *total = sums[kPlanThreads / 32 - 1];
    __syncthreads();
    return before + inclusive - value;
}

// One CTA: its time is a chain of dependent loads (ids, lengths, last pages, their counts; the
// free pages' counts are read ahead), so what an entry needs stays in shared memory up to
// kPlanThreads entries.  workspace: found [num_pages] | first [n] | source [n] | target [n].
__global__ void __launch_bounds__(kPlanThreads) extend_kernel(Kv4View view, const int32_t* __restrict__ seqs, int n,
                                                              const int32_t* __restrict__ counts, int count,
                                                              int32_t* __restrict__ workspace) {
    __shared__ int32_t ids[kMostEntries];
    __shared__ int32_t near[3][kPlanThreads];
    __shared__ int short_of_columns;
    pdl_wait();
    pdl_launch_dependents();
    int32_t* found = workspace;
    const bool few = n <= kPlanThreads;
    int32_t* first = few ? near[0] : found + view.num_pages;
    int32_t* needs = few ? near[1] : found + view.num_pages + 2 * n;
    int32_t* copies = few ? near[2] : found + view.num_pages + n;
    int32_t* source = found + view.num_pages + n;
    int32_t* target = source + n;
    const int size = view.page_size();
    int refs_ahead = threadIdx.x < view.num_pages ? view.refs[threadIdx.x] : 1;
    const int status = threadIdx.x == 0 ? view.status[0] : 0;
    for (int i = threadIdx.x; i < n; i += kPlanThreads) ids[i] = seqs[i];
    // After an extend that found no room none succeeds until the caller has seen it: the tokens in between would be
    // missing from the sequence.
    if (threadIdx.x == 0) short_of_columns = status & kKv4StatusFull;
    __syncthreads();

    // Pages that each entry needs: those its tokens reach, and one for the copy of
    // a last page that is partly filled and shared.
    int needed = 0;
    for (int base = 0; base < n; base += kPlanThreads) {
        const int i = base + threadIdx.x;
        int need = 0, copied = -1;
        if (i < n) {
            if (first_of(view, ids, i)) {
                const int s = ids[i], held = view.length_of(s);
                const int more = max(0, counts ? counts[i] : count);
                // 64 bits: a count near the int limit must not wrap past the check.
                const int64_t columns = (static_cast<int64_t>(held) + more + size - 1) >> view.page_shift;
                if (columns > view.max_pages) {
                    short_of_columns = 1;
                } else {
                    need = static_cast<int>(columns) - view.pages_of(held);
                    if (more > 0 && (held & (size - 1))) {
                        const int last = view.page_at(s, held - 1);
                        if (last >= 0 && view.refs[last] > 1) {
                            copied = last;
                            ++need;
                        }
                    }
                }
            } else {
                need = -1;
                if (ids[i] != -1) atomicOr(view.status, kKv4StatusSequence);
            }
        }
        // 64 bits: 1024 entries may need 2^26 pages each.  Past the pool's end the first pages do not matter.
        const int64_t most = view.num_pages + 1ll;
        int64_t total;
        const int64_t before = block_scan(static_cast<int64_t>(max(need, 0)), &total);
        if (i < n) {
            first[i] = static_cast<int>(min(needed + before, most));
            copies[i] = copied;
            needs[i] = need;  // -1: not an entry to extend
        }
        needed = static_cast<int>(min(needed + total, most));
    }

    // The lowest free pages, in order.
    int free_pages = 0;
    for (int base = 0; base < view.num_pages && free_pages < needed; base += kPlanThreads) {
        const int p = base + threadIdx.x, next = p + kPlanThreads;
        const bool is_free = refs_ahead == 0;
        refs_ahead = next < view.num_pages ? view.refs[next] : 1;
        int total;
        const int at = free_pages + block_scan<int>(is_free, &total);
        if (is_free && at < needed) found[at] = p;
        free_pages += total;
    }
    __syncthreads();
    if (short_of_columns || free_pages < needed) {  // all or nothing, and no writes until the bit is cleared
        for (int i = threadIdx.x; i < n; i += kPlanThreads) source[i] = -1;
        if (threadIdx.x == 0) atomicOr(view.status, kKv4StatusFull);
        return;
    }

    // Hand them out, a warp per entry.
    for (int i = threadIdx.x >> 5; i < n; i += kPlanThreads / 32) {
        const int lane = threadIdx.x & 31;
        const int need = needs[i], at = first[i], copied = copies[i];
        const int s = ids[i];
        __syncwarp();
        if (lane == 0) {
            source[i] = need < 0 ? -1 : copied;
            if (copied >= 0) target[i] = found[at];
        }
        if (need < 0) continue;
        const int held = view.length_of(s), more = max(0, counts ? counts[i] : count);
        int column = view.pages_of(held) - (copied >= 0);
        for (int j = lane; j < need; j += 32) {
            const int page = found[at + j];
            view.table[static_cast<int64_t>(s) * view.max_pages + column + j] = page;
            view.refs[page] = 1;
        }
        if (lane == 0 && copied >= 0) atomicSub(view.refs + copied, 1);
        __syncwarp();
        if (lane == 0) view.lengths[s] = held + more;
    }
}

// fork, first half, entry i: the parent's row as it is, and a reference more for each page.
__device__ void fork_read(const Kv4View& view, const int32_t* parents, const int32_t* children, int n, int i, int thread,
                          int threads, int32_t* workspace) {
    const int parent = parents[i];
    const bool fine = view.has_sequence(parent) && first_of(view, children, i);
    if (thread == 0) {
        workspace[i] = fine ? view.length_of(parent) : -1;
        if (!fine && children[i] != -1) atomicOr(view.status, kKv4StatusSequence);
    }
    if (!fine) return;
    int32_t* row = workspace + n + static_cast<int64_t>(i) * view.max_pages;
    const int pages = view.pages_of(view.length_of(parent));
    for (int j = thread; j < pages; j += threads) {
        const int page = view.table[static_cast<int64_t>(parent) * view.max_pages + j];
        row[j] = page;
        if (page >= 0 && page < view.num_pages) atomicAdd(view.refs + page, 1);
    }
}

// fork, second half: the child gives its pages back and takes the row read.  Its length is
// written by the caller, after every thread has read the old one.
__device__ void fork_write(const Kv4View& view, const int32_t* children, int n, int i, int thread, int threads,
                           const int32_t* workspace) {
    const int length = workspace[i];
    if (length < 0) return;
    const int child = children[i];
    const int before = view.pages_of(view.length_of(child)), after = view.pages_of(length);
    const int32_t* row = workspace + n + static_cast<int64_t>(i) * view.max_pages;
    int32_t* to = view.table + static_cast<int64_t>(child) * view.max_pages;
    for (int j = thread; j < max(before, after); j += threads) {
        if (j < before) {
            const int page = to[j];
            if (page >= 0 && page < view.num_pages) atomicSub(view.refs + page, 1);
        }
        to[j] = j < after ? row[j] : -1;
    }
}

// Both halves in one CTA, a warp per entry.
__global__ void __launch_bounds__(kPlanThreads) fork_kernel(Kv4View view, const int32_t* __restrict__ parents,
                                                            const int32_t* __restrict__ children, int n,
                                                            int32_t* __restrict__ workspace) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = warp; i < n; i += kPlanThreads / 32) fork_read(view, parents, children, n, i, lane, 32, workspace);
    __syncthreads();
    for (int i = warp; i < n; i += kPlanThreads / 32) fork_write(view, children, n, i, lane, 32, workspace);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if (workspace[i] >= 0) view.lengths[children[i]] = workspace[i];
}

__global__ void __launch_bounds__(kRowThreads) fork_read_kernel(Kv4View view, const int32_t* __restrict__ parents,
                                                                const int32_t* __restrict__ children, int n,
                                                                int32_t* __restrict__ workspace) {
    pdl_wait();
    pdl_launch_dependents();
    fork_read(view, parents, children, n, blockIdx.x, threadIdx.x, kRowThreads, workspace);
}

__global__ void __launch_bounds__(kRowThreads) fork_write_kernel(Kv4View view, const int32_t* __restrict__ children,
                                                                 int n, const int32_t* __restrict__ workspace) {
    pdl_wait();
    pdl_launch_dependents();
    fork_write(view, children, n, blockIdx.x, threadIdx.x, kRowThreads, workspace);
    __syncthreads();
    if (threadIdx.x == 0 && workspace[blockIdx.x] >= 0) view.lengths[children[blockIdx.x]] = workspace[blockIdx.x];
}

__global__ void __launch_bounds__(kRowThreads) truncate_kernel(Kv4View view, const int32_t* __restrict__ seqs,
                                                               const int32_t* __restrict__ lengths) {
    pdl_wait();
    pdl_launch_dependents();
    const int i = blockIdx.x;
    if (!first_of(view, seqs, i)) {
        if (threadIdx.x == 0 && seqs[i] != -1) atomicOr(view.status, kKv4StatusSequence);
        return;
    }
    const int s = seqs[i], held = view.length_of(s);
    const int kept = lengths ? min(held, max(0, lengths[i])) : 0;
    int32_t* row = view.table + static_cast<int64_t>(s) * view.max_pages;
    for (int j = view.pages_of(kept) + threadIdx.x; j < view.pages_of(held); j += kRowThreads) {
        const int page = row[j];
        if (page >= 0 && page < view.num_pages) atomicSub(view.refs + page, 1);
        row[j] = -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) view.lengths[s] = kept;
}

// One CTA.  workspace: source [num_pages] | target [num_pages] | place [num_pages].
__global__ void __launch_bounds__(kPlanThreads) compact_kernel(Kv4View view, int32_t* __restrict__ workspace) {
    pdl_wait();
    pdl_launch_dependents();
    int32_t* source = workspace;
    int32_t* target = source + view.num_pages;
    int32_t* place = target + view.num_pages;
    int live = 0;
    for (int base = 0; base < view.num_pages; base += kPlanThreads) {
        const int p = base + threadIdx.x;
        int total;
        block_scan<int>(p < view.num_pages && view.refs[p] > 0, &total);
        live += total;
    }
    int moved = 0, holes = 0;
    for (int base = 0; base < view.num_pages; base += kPlanThreads) {
        const int p = base + threadIdx.x;
        const bool used = p < view.num_pages && view.refs[p] > 0;
        const bool moves = used && p >= live, hole = p < live && !used;
        int total;
        const int at = moved + block_scan<int>(moves, &total);
        moved += total;
        const int into = holes + block_scan<int>(hole, &total);
        holes += total;
        if (moves) source[at] = p;
        if (hole) target[into] = p;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < moved; i += kPlanThreads) {
        place[source[i]] = target[i];
        view.refs[target[i]] = view.refs[source[i]];
        view.refs[source[i]] = 0;
    }
    if (threadIdx.x == 0) {
        view.status[1] = live;
        view.status[2] = moved;
    }
}

__global__ void __launch_bounds__(kRowThreads) place_kernel(Kv4View view, const int32_t* __restrict__ workspace) {
    pdl_wait();
    pdl_launch_dependents();
    const int s = blockIdx.x;
    const int live = view.status[1];
    const int32_t* place = workspace + 2 * static_cast<int64_t>(view.num_pages);
    const int pages = view.pages_of(view.length_of(s));
    for (int j = threadIdx.x; j < pages; j += kRowThreads) {
        const int64_t at = static_cast<int64_t>(s) * view.max_pages + j;
        const int page = view.table[at];
        if (page >= live && page < view.num_pages) view.table[at] = place[page];
    }
}

// A persistent grid over (entry, layer, part of the page); a thread has kUnits 16-byte loads in
// flight.  Bound by HBM: a copy of 0.5 GB runs at what the device's plain copy reaches.
constexpr int kUnits = 8;

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(Kv4View view, const int32_t* __restrict__ sources,
                                                            const int32_t* __restrict__ targets, int64_t count,
                                                            const int32_t* __restrict__ count_dev) {
    pdl_wait();
    pdl_launch_dependents();
    if (count_dev) count = min(count, static_cast<int64_t>(*count_dev));
    const int units = static_cast<int>(view.page_bytes / 16);
    constexpr int kPart = kCopyThreads * kUnits;
    const int parts = (units + kPart - 1) / kPart;
    const int64_t items = count * view.layers * parts;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t of_page = item / parts;
        const int part = static_cast<int>(item - of_page * parts);
        const int64_t entry = of_page / view.layers;
        const int layer_number = static_cast<int>(of_page - entry * view.layers);
        const int from = sources[entry], to = targets[entry];
        if (from < 0 || from >= view.num_pages || to < 0 || to >= view.num_pages) continue;
        uint8_t* layer = view.pages + layer_number * view.layer_bytes;
        const auto* src = reinterpret_cast<const uint4*>(layer + from * view.page_bytes);
        auto* dst = reinterpret_cast<uint4*>(layer + to * view.page_bytes);
        uint4 v[kUnits];
        const int first = part * kPart + threadIdx.x;
#pragma unroll
        for (int i = 0; i < kUnits; ++i)
            if (first + i * kCopyThreads < units) v[i] = __ldcs(src + first + i * kCopyThreads);
#pragma unroll
        for (int i = 0; i < kUnits; ++i)
            if (first + i * kCopyThreads < units) __stcs(dst + first + i * kCopyThreads, v[i]);
    }
}

}  // namespace

int kv4_copy_launch(const char* what, const Kv4View& view, const int32_t* sources, const int32_t* targets,
                    int64_t count, const int32_t* count_dev, cudaStream_t stream) {
    if (count == 0) return POPKV_OK;
    constexpr int64_t kGrid = 148 * 6;
    const int64_t units = view.page_bytes / 16, part = kCopyThreads * kUnits;
    const int64_t items = count * view.layers * ((units + part - 1) / part);
    const cudaError_t err = launch_pdl(copy_kernel, dim3(static_cast<unsigned>(items < kGrid ? items : kGrid)),
                                       dim3(kCopyThreads), 0, stream, 1, view, sources, targets, count, count_dev);
    if (err != cudaSuccess) return fail(POPKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
    return check_launch(what);
}

}  // namespace popkv

extern "C" int popkv_kv4_copy_pages(const popkv_kv4_cache* cache, const int32_t* sources, const int32_t* targets,
                                    int64_t count, void* stream) {
    using namespace popkv;
    Kv4View view;
    if (int status = kv4_view("popkv_kv4_copy_pages", cache, &view)) return status;
    if (count < 0 || count > (1 << 30)) return fail(POPKV_ERR_INVALID, "popkv_kv4_copy_pages: count out of range");
    if (count == 0) return POPKV_OK;
    if (!sources || !targets) return fail(POPKV_ERR_INVALID, "popkv_kv4_copy_pages: null pointer");
    return kv4_copy_launch("popkv_kv4_copy_pages", view, sources, targets, count, nullptr,
                           static_cast<cudaStream_t>(stream));
}

namespace popkv {
namespace {
template <typename... Parameters, typename... Arguments>
int launch_plan(const char* what, void (*kernel)(Parameters...), unsigned blocks, int threads, void* stream,
                Arguments... arguments) {
    const cudaError_t err =
        launch_pdl(kernel, dim3(blocks), dim3(threads), 0, static_cast<cudaStream_t>(stream), 1, arguments...);
    if (err != cudaSuccess) return fail(POPKV_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
    return check_launch(what);
}

int check_entries(const char* what, int64_t n) {
    if (n < 0 || n > kMostEntries)
        return fail(POPKV_ERR_INVALID, "%s: between 0 and 4096 sequences in one call", what);
    return POPKV_OK;
}
}  // namespace
}  // namespace popkv

extern "C" int popkv_kv4_extend(const popkv_kv4_cache* cache, const int32_t* seqs, int64_t n, const int32_t* counts,
                                int64_t count, int32_t* workspace, void* stream) {
    using namespace popkv;
    Kv4View view;
    if (int status = kv4_view("popkv_kv4_extend", cache, &view)) return status;
    if (int status = check_entries("popkv_kv4_extend", n)) return status;
    if (count < 0 || count > (1 << 30)) return fail(POPKV_ERR_INVALID, "popkv_kv4_extend: count out of range");
    if (n == 0) return POPKV_OK;
    if (!seqs || !workspace) return fail(POPKV_ERR_INVALID, "popkv_kv4_extend: null pointer");
    const auto s = static_cast<cudaStream_t>(stream);
    if (int status = launch_plan("popkv_kv4_extend", extend_kernel, 1, kPlanThreads, stream, view, seqs,
                                 static_cast<int>(n), counts, static_cast<int>(count), workspace))
        return status;
    const int32_t* source = workspace + view.num_pages + n;
    return kv4_copy_launch("popkv_kv4_extend", view, source, source + n, n, nullptr, s);
}

extern "C" int popkv_kv4_fork(const popkv_kv4_cache* cache, const int32_t* parents, const int32_t* children,
                              int64_t n, int32_t* workspace, void* stream) {
    using namespace popkv;
    Kv4View view;
    if (int status = kv4_view("popkv_kv4_fork", cache, &view)) return status;
    if (int status = check_entries("popkv_kv4_fork", n)) return status;
    if (n == 0) return POPKV_OK;
    if (!parents || !children || !workspace) return fail(POPKV_ERR_INVALID, "popkv_kv4_fork: null pointer");
    const int count = static_cast<int>(n);
    const char* what = "popkv_kv4_fork";
    // One CTA for both halves while the rows are few (one launch less), a CTA per row beyond.
    if (n * view.max_pages <= 32768)
        return launch_plan(what, fork_kernel, 1, kPlanThreads, stream, view, parents, children, count, workspace);
    if (int status = launch_plan(what, fork_read_kernel, count, kRowThreads, stream, view, parents, children, count,
                                 workspace))
        return status;
    return launch_plan(what, fork_write_kernel, count, kRowThreads, stream, view, children, count,
                       static_cast<const int32_t*>(workspace));
}

extern "C" int popkv_kv4_truncate(const popkv_kv4_cache* cache, const int32_t* seqs, int64_t n,
                                  const int32_t* lengths, void* stream) {
    using namespace popkv;
    Kv4View view;
    if (int status = kv4_view("popkv_kv4_truncate", cache, &view)) return status;
    if (int status = check_entries("popkv_kv4_truncate", n)) return status;
    if (n == 0) return POPKV_OK;
    if (!seqs) return fail(POPKV_ERR_INVALID, "popkv_kv4_truncate: null pointer");
    return launch_plan("popkv_kv4_truncate", truncate_kernel, static_cast<unsigned>(n), kRowThreads, stream, view, seqs,
                       lengths);
}

extern "C" int popkv_kv4_compact(const popkv_kv4_cache* cache, int32_t* workspace, void* stream) {
    using namespace popkv;
    Kv4View view;
    if (int status = kv4_view("popkv_kv4_compact", cache, &view)) return status;
    if (!workspace) return fail(POPKV_ERR_INVALID, "popkv_kv4_compact: null pointer");
    const char* what = "popkv_kv4_compact";
    if (int status = launch_plan(what, compact_kernel, 1, kPlanThreads, stream, view, workspace)) return status;
    if (int status = launch_plan(what, place_kernel, static_cast<unsigned>(view.max_seqs), kRowThreads, stream, view,
                                 static_cast<const int32_t*>(workspace)))
        return status;
    return kv4_copy_launch(what, view, workspace, workspace + view.num_pages, view.num_pages, view.status + 2,
                           static_cast<cudaStream_t>(stream));
}
