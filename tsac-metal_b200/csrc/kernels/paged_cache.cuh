// Paged key/value cache: device view and launches (paged_cache.cu).  The
// layout and the meaning of each operation are stated in include/tsac_cuda.h.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace tsacb::dev
{
constexpr int CACHE_MAX_LIST = 4096;       // sequences named by one call
constexpr int CACHE_MAX_SEQUENCES = 65536; // one bit each in the duplicate check

struct CacheView
{
    unsigned char* pool; // [planes][pages][page_size][row_bytes], planes = layers x {keys, values}
    int* tables;         // [sequences][max_pages]
    int* counts;         // [sequences] pages held
    int* lengths;        // [sequences] positions committed
    int* refs;           // [pages] table entries that name the page; 0 = free
    long long plane_bytes;
    int planes, pages, page_shift, row_bytes, sequences, max_pages;

    __host__ __device__ int page_size() const { return 1 << page_shift; }
    __host__ __device__ long long page_bytes() const { return static_cast<long long>(row_bytes) << page_shift; }
};

// Page of table entry `page` of a sequence; -1 when the entry is not held or
// does not name a page of the pool, so that no caller indexes with it.
__device__ __forceinline__ int cache_page(const CacheView& c, int sequence, int held, int entry)
{
    if (entry < 0 || entry >= held)
        return -1;
    const int p = c.tables[static_cast<size_t>(sequence) * c.max_pages + entry];
    return static_cast<unsigned>(p) < static_cast<unsigned>(c.pages) ? p : -1;
}

// Pages a sequence holds, within its table's width whatever the count says.
__device__ __forceinline__ int cache_held(const CacheView& c, int sequence)
{
    const int n = c.counts[sequence];
    return n < 0 ? 0 : (n < c.max_pages ? n : c.max_pages);
}

// Sequence of list entry i (the list may be absent: entry i is sequence i);
// -1 when it is not a sequence of the cache.
__device__ __forceinline__ int cache_sequence(const CacheView& c, const int* sequences, int i)
{
    const int s = sequences ? sequences[i] : i;
    return static_cast<unsigned>(s) < static_cast<unsigned>(c.sequences) ? s : -1;
}

size_t cache_reserve_scratch(size_t count, size_t slots);
void cache_reserve(const CacheView& c, const int* sequences, const int* positions, int count, int slots,
                   void* scratch, unsigned* error_word, cudaStream_t stream);
void cache_fork(const CacheView& c, const int* parents, const int* children, int count, unsigned* error_word,
                cudaStream_t stream);
void cache_release(const CacheView& c, const int* sequences, const int* positions, int count, unsigned* error_word,
                   cudaStream_t stream);

struct AppendRows
{
    const unsigned char* source[2];         // keys, values
    long long batch_bytes[2], node_bytes[2], head_bytes[2];
    int head_chunks;                        // 16-byte chunks of one head
    int heads;
};
void cache_append(const CacheView& c, int layer, const AppendRows& rows, const int* sequences, const int* nodes,
                  const int* starts, int count, int max_nodes, unsigned* error_word, cudaStream_t stream);
void cache_keep(const CacheView& c, const int* sequences, const int* path, const int* accepted, const int* starts,
                int* lengths_out, int count, int width, unsigned* error_word, cudaStream_t stream);

size_t cache_compact_scratch(size_t pages);
void cache_compact(const CacheView& c, int* tables_out, int* refs_out, int* live, void* scratch,
                   unsigned* error_word, cudaStream_t stream);
} // namespace tsacb::dev
