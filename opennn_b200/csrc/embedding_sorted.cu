// Gradient of the embedding table, summed by token in a fixed order:
//   dW[v, :] (+)= sqrt(E) * sum over the positions n with id v of (dY + dY2)[n, :],   0 < v < V.
// No atomics on floating-point values: the same inputs give the same bits.
//
// Bound by HBM: every gradient row is read once and every table row written once.
//   1  the positions are sorted by id.  CTA c has every P-th row of the table from the c-th on (neighbouring ids are often
//      frequent together): it reads all ids, keeps the positions of its own, counts those of the CTAs before it, which
//      tells where its part of the sorted list begins, and sorts what it has kept.  No CTA needs another's result, so one
//      launch does it: 6.5 us for 16384 positions (a radix sort by one cluster, or in launches of counts and places: 14 to
//      20);
//   2  the sorted positions are cut into equal chunks, whatever their ids, so that a frequent token is spread over many
//      CTAs; a group of threads adds the rows of a chunk, and writes the table row of each run of equal ids that lies inside it.
//      Runs that cross the edge of a chunk leave a partial sum.  Other CTAs of the same launch write the zeros of the
//      table rows that do not occur;
//   3  the partial sums of each run that crosses an edge are added in order.
// Few positions take one launch instead: every CTA owns some rows of the table and looks for their ids itself.
//
// Measured on a B200 (copy bandwidth 6.57 TB/s): 128 x 1024 positions of 1024 features and two inputs, frequencies 1/v over
// 50021 tokens, 243 us: sort 25, chunks 198 (1.28 GB: 6.5 TB/s), joins the rest.  64 x 256 positions over 32000 tokens, 43 us: 6, 30
// (173 MB: 5.8 TB/s), 6.  32 x 32 positions of 64 features and 1000 tokens: 3.3 us, 7 at frequencies 1/v.
#include "common.cuh"
#include "launch_counter.h"

namespace onn
{

namespace
{

// ---------------------------------------------------------------------------------------
// Few positions
// ---------------------------------------------------------------------------------------

constexpr int kOwnerThreads = 256;
constexpr int kOwnerWarps = kOwnerThreads / 32;
constexpr int kTile = 1024;                       // ids looked at together
constexpr int kOwnerColumns = 64;
constexpr int kOwnerGroups = kOwnerThreads / kOwnerColumns;
constexpr int kOwnerInFlight = 16;                // gradient elements a thread has under way, of one input at a time
constexpr int kMaxOwned = 32;                     // rows of a CTA, summed in shared memory

// CTA (x, y) owns `owned` consecutive rows of the table, 64 columns of them.  It walks over all ids in order and keeps those that
// are its own (in order: prefix sums); four groups of 64 threads, one per column, add every fourth of their gradient
// rows each, and the groups' sums are added in order.
__global__ void __launch_bounds__(kOwnerThreads, 3)
embedding_owner_kernel(const float* __restrict__ ids, const float* __restrict__ dY, const float* __restrict__ dY2,
                       float* __restrict__ dW, int tokens, int E, int V, float scale, int owned, int accumulate)
{
    __shared__ float sums[kOwnerGroups][kMaxOwned][kOwnerColumns];
    __shared__ unsigned char present[kMaxOwned];
    __shared__ unsigned short list_row[kTile];
    __shared__ unsigned short list_token[kTile];
    __shared__ int warp_count[kOwnerWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = tid / kOwnerColumns, in_group = tid % kOwnerColumns;
    const int v0 = blockIdx.x * owned, v1 = min(v0 + owned, V);
    const int column = blockIdx.y * kOwnerColumns + in_group;
    for(int r = 0; r < owned; r++) sums[group][r][in_group] = 0.f;
    if(tid < kMaxOwned) present[tid] = 0;
    for(int first = 0; first < tokens; first += kTile)
    {
        constexpr int kEach = kTile / kOwnerThreads;
        int found[kEach];
        int mine = 0;
#pragma unroll
        for(int k = 0; k < kEach; k++)
        {
            const int n = first + tid * kEach + k;
            const long long v = n < tokens ? token_index(__ldg(ids + n)) : 0;
            found[k] = v > 0 && v >= v0 && v < v1 ? (int)v - v0 : -1;
            mine += found[k] >= 0;
        }
        int before = mine;
#pragma unroll
        for(int offset = 1; offset < 32; offset <<= 1)
        {
            const int other = __shfl_up_sync(0xffffffffu, before, offset);
            if(lane >= offset) before += other;
        }
        __syncthreads();                               // the lists of the tile before have been read
        if(lane == 31) warp_count[warp] = before;
        __syncthreads();
        before -= mine;
        int total = 0;
#pragma unroll
        for(int w = 0; w < kOwnerWarps; w++)
        {
            if(w < warp) before += warp_count[w];
            total += warp_count[w];
        }
#pragma unroll
        for(int k = 0; k < kEach; k++)
        {
            if(found[k] < 0) continue;
            list_row[before] = (unsigned short)found[k];
            list_token[before] = (unsigned short)(tid * kEach + k);
            present[found[k]] = 1;
            before++;
        }
        __syncthreads();
        if(column < E)
        {
            // equal ids one after the other are added in a register
            int current = -1;
            float sum = 0.f;
            for(int i = group; i < total; i += kOwnerGroups * kOwnerInFlight)
            {
                float g[kOwnerInFlight];
                int at[kOwnerInFlight];
#pragma unroll
                for(int k = 0; k < kOwnerInFlight; k++)
                {
                    const int j = i + k * kOwnerGroups;
                    at[k] = first + (j < total ? list_token[j] : 0);
                    g[k] = j < total ? __ldg(dY + (long long)at[k] * E + column) : 0.f;
                }
                if(dY2)
                {
#pragma unroll
                    for(int k = 0; k < kOwnerInFlight; k++)
                        if(i + k * kOwnerGroups < total) g[k] += __ldg(dY2 + (long long)at[k] * E + column);
                }
#pragma unroll
                for(int k = 0; k < kOwnerInFlight; k++)
                {
                    const int j = i + k * kOwnerGroups;
                    if(j >= total) break;
                    const int row = list_row[j];
                    if(row != current)
                    {
                        if(current >= 0) sums[group][current][in_group] += sum;
                        current = row;
                        sum = 0.f;
                    }
                    sum += g[k];
                }
            }
            if(current >= 0) sums[group][current][in_group] += sum;
        }
    }
    __syncthreads();
    if(column >= E) return;
    auto sum_of = [&](int r)
    {
        float sum = sums[0][r][in_group];
#pragma unroll
        for(int q = 1; q < kOwnerGroups; q++) sum += sums[q][r][in_group];
        return sum * scale;
    };
    float* const to = dW + (long long)v0 * E + column;
    if(!accumulate)
    {
        for(int r = group; r < v1 - v0; r += kOwnerGroups) to[(long long)r * E] = sum_of(r);
        return;
    }
    // the rows' earlier values are asked for together
    constexpr int kRows = kMaxOwned / kOwnerGroups;
    float earlier[kRows];
#pragma unroll
    for(int k = 0; k < kRows; k++)
    {
        const int r = group + k * kOwnerGroups;
        earlier[k] = r < v1 - v0 && present[r] ? to[(long long)r * E] : 0.f;
    }
#pragma unroll
    for(int k = 0; k < kRows; k++)
    {
        const int r = group + k * kOwnerGroups;
        if(r < v1 - v0 && present[r]) to[(long long)r * E] = earlier[k] + sum_of(r);
    }
}

// ---------------------------------------------------------------------------------------
// 1: sort
// ---------------------------------------------------------------------------------------

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMinParts = 128;                    // CTAs: a power of two
constexpr int kMaxRows = 512;                     // of the table, a CTA's part
constexpr int kRowBits = 9;
constexpr int kList = 512;                        // positions that a warp keeps; beyond that it reads the ids again

struct SortShared
{
    unsigned int count[kSortWarps][kMaxRows];     // of each warp: how often a row occurs; then where its next position goes
    unsigned int position[kSortWarps][kList];
    unsigned short row[kSortWarps][kList];
    unsigned short place[kSortWarps][kList];      // among the warp's positions of the same row
    unsigned int warp_sum[kSortWarps];
    unsigned int warp_lower[kSortWarps];
};

// The lanes of the warp whose row is this lane's: one vote per bit.
__device__ __forceinline__ unsigned int lanes_with(unsigned int row, bool there)
{
    unsigned int same = __ballot_sync(0xffffffffu, there);
#pragma unroll
    for(int b = 0; b < kRowBits; b++)
    {
        const unsigned int set = __ballot_sync(0xffffffffu, (row >> b) & 1u);
        same &= (row >> b) & 1u ? set : ~set;
    }
    return same;
}

// CTA c has the rows v of the table with (v - 1) % parts = c, parts = 1 << part_bits; its row r is v = (r << part_bits) + c + 1.
// Warp w looks at the w-th of 32 equal stretches of the ids.  present[v] says whether v occurs.
__global__ void __launch_bounds__(kSortThreads, 1)
embedding_sort_kernel(const float* __restrict__ ids, uint2* __restrict__ sorted, int* __restrict__ control,
                      unsigned char* __restrict__ present, int tokens, int V, int part_bits)
{
    extern __shared__ __align__(16) unsigned char bytes[];
    SortShared& shared = *reinterpret_cast<SortShared*>(bytes);
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned int below = (1u << lane) - 1u;
    const unsigned int part = blockIdx.x, part_mask = (1u << part_bits) - 1u;
    const int rows = V - 1 > (int)part ? ((V - 2 - (int)part) >> part_bits) + 1 : 0;
    constexpr int kBlock = 512;                       // ids a warp looks at together, 16 neighbouring ones per lane
    const long long stretch = ((tokens + kSortWarps - 1) / kSortWarps + kBlock - 1) / kBlock * kBlock;
    const long long from = warp * stretch < tokens ? warp * stretch : tokens, to = from + stretch < tokens ? from + stretch : tokens;
    const bool vec = aligned16(ids);
    unsigned int* const count = shared.count[warp];
    unsigned int* const list_position = shared.position[warp];
    unsigned short* const list_row = shared.row[warp];
    unsigned short* const list_place = shared.place[warp];
    for(int r = lane; r < rows; r += 32) count[r] = 0;

    // found(n of the lane's first id, a bit for each of its ids that is one of this CTA's, how many of the warp's lie before the
    // lane's, how many there are)
    unsigned int lower = 0;
    auto scan = [&](auto found)
    {
        for(long long first = from; first < to; first += kBlock)
        {
            const long long n = first + lane * 16;
            // 2^23 + id, rounded toward zero, holds trunc(id) in its low bits for 0 <= id < 2^23; everything else (negative, larger,
            // NaN) comes out far above V - 1 when 2^23 + 1 is taken from the bits
            unsigned int mine = 0;
            auto look = [&](float id, int j)
            {
                const unsigned int before = __float_as_uint(__fadd_rz(id, 8388608.f)) - 0x4b000001u;      // id - 1
                const unsigned int its = before < (unsigned int)(V - 1) ? before & part_mask : 0xffffffffu;
                lower += its < part;
                mine |= its == part ? 1u << j : 0u;
            };
            if(vec && n + 16 <= to)
            {
#pragma unroll
                for(int q = 0; q < 4; q++)
                {
                    const float4 f = __ldg(reinterpret_cast<const float4*>(ids + n) + q);
                    look(f.x, q * 4); look(f.y, q * 4 + 1); look(f.z, q * 4 + 2); look(f.w, q * 4 + 3);
                }
            }
            else
            {
                for(int j = 0; j < 16 && n + j < to; j++) look(__ldg(ids + n + j), j);
            }
            if(!__any_sync(0xffffffffu, mine != 0)) continue;
            int upto = __popc(mine);
#pragma unroll
            for(int offset = 1; offset < 32; offset <<= 1)
            {
                const int other = __shfl_up_sync(0xffffffffu, upto, offset);
                if(lane >= offset) upto += other;
            }
            found((unsigned int)n, mine, upto - __popc(mine), __shfl_sync(0xffffffffu, upto, 31));
        }
    };
    auto keep = [&](unsigned int n, unsigned int mine, int at)
    {
        for(; mine != 0; mine &= mine - 1, at++)
        {
            if(at >= kList) break;
            const unsigned int position = n + __ffs(mine) - 1;
            list_position[at] = position;
            list_row[at] = (unsigned short)((__float_as_uint(__fadd_rz(__ldg(ids + position), 8388608.f)) - 0x4b000001u) >> part_bits);
        }
    };
    int kept = 0;
    scan([&](unsigned int n, unsigned int mine, int before, int all) { keep(n, mine, kept + before); kept += all; });
    __syncwarp();
    // act(whether there is one, its row, position, index on the list) for the warp's positions in order, 32 at a time: from its
    // list, or, where it is too short, from the ids again, 512 of them by way of the list
    const bool listed = kept <= kList;
    auto each = [&](auto act)
    {
        auto from_list = [&](int n)
        {
            for(int i = lane; i - lane < n; i += 32)
            {
                const bool there = i < n;
                act(there, there ? list_row[i] : 0u, there ? list_position[i] : 0u, i);
            }
        };
        if(listed) from_list(kept);
        else
        {
            scan([&](unsigned int n, unsigned int mine, int before, int all)
            {
                keep(n, mine, before);
                __syncwarp();
                from_list(all);
                __syncwarp();
            });
        }
    };
    const unsigned int lower_of_warp = __reduce_add_sync(0xffffffffu, lower);
    if(lane == 0) shared.warp_lower[warp] = lower_of_warp;
    // the place of a position among the warp's of its row, which count[row] counts up
    auto next_place = [&](bool there, unsigned int row)
    {
        const unsigned int same = lanes_with(row, there);
        const unsigned int place = there ? count[row] + __popc(same & below) : 0u;
        __syncwarp();
        if(there && (same & below) == 0) count[row] += __popc(same);
        __syncwarp();
        return place;
    };
    each([&](bool there, unsigned int row, unsigned int, int i)
    {
        const unsigned int place = next_place(there, row);
        if(listed && there) list_place[i] = (unsigned short)place;
    });
    __syncthreads();

    // thread r: where each warp's share of row r goes
    unsigned int all = 0;
    if(tid < rows)
    {
#pragma unroll 8
        for(int w = 0; w < kSortWarps; w++) all += shared.count[w][tid];
        present[(tid << part_bits) + part + 1] = all != 0;
    }
    if(tid == 0 && part == 0) present[0] = 0;
    unsigned int upto = all;
#pragma unroll
    for(int offset = 1; offset < 32; offset <<= 1)
    {
        const unsigned int other = __shfl_up_sync(0xffffffffu, upto, offset);
        if(lane >= offset) upto += other;
    }
    if(lane == 31) shared.warp_sum[warp] = upto;
    __syncthreads();
    unsigned int start = __reduce_add_sync(0xffffffffu, shared.warp_lower[lane] + (lane < warp ? shared.warp_sum[lane] : 0u)) + upto - all;
    if(tid == kSortThreads - 1 && blockIdx.x == gridDim.x - 1) { control[0] = 0; control[1] = 0; control[2] = (int)(start + all); }
    if(tid < rows)
    {
#pragma unroll 8
        for(int w = 0; w < kSortWarps; w++)
        {
            const unsigned int c = shared.count[w][tid];
            shared.count[w][tid] = start;
            start += c;
        }
    }
    __syncthreads();
    each([&](bool there, unsigned int row, unsigned int position, int i)
    {
        const unsigned int at = listed ? there ? count[row] + list_place[i] : 0u : next_place(there, row);
        if(there) sorted[at] = make_uint2((row << part_bits) + part + 1u, position);
    });
}

// ---------------------------------------------------------------------------------------
// 2: chunks, and 3: runs that cross their edges
// ---------------------------------------------------------------------------------------

constexpr int kReduceThreads = 256;
template <int VEC> struct Piece;
template <> struct Piece<4>
{
    using type = float4;
    static __device__ __forceinline__ float4 zero() { return make_float4(0.f, 0.f, 0.f, 0.f); }
    static __device__ __forceinline__ float4 load(const float* p) { return ld4_stream(p); }
    static __device__ __forceinline__ void store(float* p, float4 v) { st4(p, v); }
    static __device__ __forceinline__ float4 add(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
    static __device__ __forceinline__ float4 scaled(float4 a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }
};
template <> struct Piece<1>
{
    using type = float;
    static __device__ __forceinline__ float zero() { return 0.f; }
    static __device__ __forceinline__ float load(const float* p) { return __ldcs(p); }
    static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
    static __device__ __forceinline__ float add(float a, float b) { return a + b; }
    static __device__ __forceinline__ float scaled(float a, float s) { return a * s; }
};

template <int VEC>
__device__ __forceinline__ void put_row(float* to, typename Piece<VEC>::type sum, float scale, int accumulate)
{
    using P = Piece<VEC>;
    sum = P::scaled(sum, scale);
    if(accumulate) sum = P::add(sum, P::load(to));
    P::store(to, sum);
}

constexpr int kLongRun = 4;                       // a run that crosses more chunk edges is long

constexpr int kMaxChunk = 64;
constexpr int kTree = 8;                          // gradient rows of one token that are added in pairs
constexpr int kZeroRows = 32;                     // table rows of a CTA that writes zeros

// A warp writes a row, or a part of it a short one, in 16-byte pieces between the row's ends.
__device__ __forceinline__ void zero_absent_rows(const unsigned char* present, float* __restrict__ dW, int E, int V, long long v0)
{
    int width = 32;
    while(width > 4 && width * 2 >= E) width >>= 1;
    const int lane = threadIdx.x & (width - 1);
    for(int r = threadIdx.x / width; r < kZeroRows && v0 + r < V; r += kReduceThreads / width)
    {
        if(present[v0 + r]) continue;
        float* const row = dW + (v0 + r) * E;
        const int head = min((int)((-reinterpret_cast<intptr_t>(row)) & 15) / 4, E), pieces = (E - head) / 4, after = head + pieces * 4;
        if(lane < head) row[lane] = 0.f;
        for(int i = lane; i < pieces; i += width) st4(row + head + i * 4, make_float4(0.f, 0.f, 0.f, 0.f));
        if(lane < E - after) row[after + lane] = 0.f;
    }
}

// A group of `group` threads adds one chunk, group * VEC columns of it.  control = {short runs to join, long ones, sorted positions}.
// CTAs behind the first chunk_ctas * across write zeros; the `across` CTAs that have a chunk's columns lie side by side.
template <int VEC, bool TWO>
__global__ void __launch_bounds__(kReduceThreads, TWO ? 2 : 3)
embedding_chunk_kernel(const uint2* sorted, const unsigned char* present, const float* __restrict__ dY, const float* __restrict__ dY2,
                       float* __restrict__ dW, float* __restrict__ partial, int2* __restrict__ owners, int* control,
                       int E, int V, int chunk, int chunks, int chunk_ctas, int across, int group, float scale, int accumulate)
{
    using P = Piece<VEC>;
    using T = typename P::type;
    __shared__ uint2 items[kReduceThreads / 32][kMaxChunk];
    pdl_launch_dependents();
    pdl_wait();
    const unsigned int along = blockIdx.x / across;
    if(along >= (unsigned int)chunk_ctas)
    {
        zero_absent_rows(present, dW, E, V, (long long)(blockIdx.x - chunk_ctas * across) * kZeroRows);
        return;
    }
    const int which = threadIdx.x / group;
    const int index = along * (kReduceThreads / group) + which;
    const int tokens = control[2];
    const int column = ((blockIdx.x - along * across) * group + threadIdx.x % group) * VEC;
    const long long start = (long long)index * chunk;
    const int length = (int)(start < tokens ? (tokens - start < chunk ? tokens - start : chunk) : 0);
    for(int i = threadIdx.x % group; i < length; i += group) items[which][i] = sorted[start + i];
    __syncthreads();
    if(length == 0 || column >= E) return;
    const uint2* const item = items[which];
    // gradient rows a thread has under way: 128 bytes of each input, 16 scalars (they cost a register each)
    constexpr int kInFlight = VEC == 4 ? 8 : 16;
    const long long end = start + length;
    const unsigned int before = start > 0 ? sorted[start - 1].x : 0xffffffffu, behind = end < tokens ? sorted[end].x : 0xffffffffu;

    unsigned int current = item[0].x;
    bool starts_here = before != current;
    T sum = P::zero();
    auto finish = [&](bool ends_here)
    {
        if(starts_here && ends_here) put_row<VEC>(dW + (long long)current * E + column, sum, scale, accumulate);
        else
        {
            P::store(partial + ((long long)index * 2 + (starts_here ? 1 : 0)) * E + column, sum);
            if(starts_here && column == 0)
            {
                // whose partial sums have to be joined: short runs from the front of the list, long ones from its back
                const long long far = (long long)(index + kLongRun) * chunk;
                if(far < tokens && sorted[far].x == current) owners[chunks - 1 - atomicAdd(control + 1, 1)] = make_int2(index, (int)current);
                else owners[atomicAdd(control, 1)] = make_int2(index, (int)current);
            }
        }
    };
    for(int i = 0; i < length; i += kInFlight)
    {
        T row[kInFlight], other[kInFlight];
#pragma unroll
        for(int u = 0; u < kInFlight; u++)
        {
            row[u] = other[u] = P::zero();
            if(i + u >= length) continue;
            const long long at = (long long)item[i + u].y * E + column;
            row[u] = P::load(dY + at);
            if(TWO) other[u] = P::load(dY2 + at);
        }
#pragma unroll
        for(int u0 = 0; u0 < kInFlight; u0 += kTree)
        {
            if(TWO)
            {
#pragma unroll
                for(int u = u0; u < u0 + kTree; u++) row[u] = P::add(row[u], other[u]);
            }
            if(i + u0 + kTree <= length && item[i + u0].x == current && item[i + u0 + kTree - 1].x == current)
            {
                // eight of a run: in pairs, for a smaller rounding error where runs are long
#pragma unroll
                for(int d = 1; d < kTree; d *= 2)
                {
#pragma unroll
                    for(int u = u0; u < u0 + kTree; u += 2 * d) row[u] = P::add(row[u], row[u + d]);
                }
                sum = P::add(sum, row[u0]);
                continue;
            }
#pragma unroll
            for(int u = u0; u < u0 + kTree; u++)
            {
                if(i + u >= length) break;
                const unsigned int v = item[i + u].x;
                if(v != current)
                {
                    finish(true);
                    current = v;
                    starts_here = true;
                    sum = P::zero();
                }
                sum = P::add(sum, row[u]);
            }
        }
    }
    finish(behind != current);
}

// A run that starts in one chunk and goes on in the next ones: the second partial of its first chunk, then the first of each
// following one.  A CTA adds 32 * VEC columns of a long run: its eight warps take every eighth part, and their sums are added
// in order.  A warp adds a short one, four blocks of 32 * VEC columns at a time.  Short ones
// are dealt out from the first CTA on, long ones from the last, so that few CTAs have both.
template <int VEC>
__global__ void __launch_bounds__(kReduceThreads)
embedding_join_kernel(const uint2* sorted, const float* partial, const int2* owners, const int* control, float* __restrict__ dW,
                      int E, int chunk, int chunks, float scale, int accumulate)
{
    using P = Piece<VEC>;
    using T = typename P::type;
    constexpr int kWarps = kReduceThreads / 32;
    __shared__ T warp_sums[kWarps][32];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int blocks = (E + 32 * VEC - 1) / (32 * VEC), tokens = control[2];
    // part 0 of a run is its first chunk's, part j that of the j-th behind it
    auto part = [&](int index, int j, int column) { return P::load(partial + ((long long)(index + j) * 2 + (j == 0 ? 1 : 0)) * E + column); };

    const int long_runs = control[1];
    int run = (int)(gridDim.x - 1 - blockIdx.x) / blocks, block = (int)(gridDim.x - 1 - blockIdx.x) % blocks;
    for(; run < long_runs; run += (int)gridDim.x / blocks)
    {
        const int2 owner = owners[chunks - 1 - run];
        const int index = owner.x, column = (block * 32 + lane) * VEC;
        const unsigned int v = (unsigned int)owner.y;
        int parts = 1;
        while(true)
        {
            // the chunks that begin with the same id lie side by side
            const long long at = (long long)(index + parts + tid) * chunk;
            const int here = __syncthreads_count(at < tokens && sorted[at].x == v);
            parts += here;
            if(here < kReduceThreads) break;
        }
        T sum = P::zero();
        if(column < E)
        {
            for(int j = warp; j < parts; j += 8 * kWarps)
            {
                T some[8];
#pragma unroll
                for(int k = 0; k < 8; k++) some[k] = j + k * kWarps < parts ? part(index, j + k * kWarps, column) : P::zero();
#pragma unroll
                for(int k = 0; k < 8; k++) sum = P::add(sum, some[k]);
            }
        }
        warp_sums[warp][lane] = sum;
        __syncthreads();
        if(warp == 0 && column < E)
        {
            sum = warp_sums[0][lane];
#pragma unroll
            for(int q = 1; q < kWarps; q++) sum = P::add(sum, warp_sums[q][lane]);
            put_row<VEC>(dW + (long long)v * E + column, sum, scale, accumulate);
        }
        block += (int)gridDim.x % blocks;
        if(block >= blocks) { block -= blocks; run++; }
        __syncthreads();
    }

    const int short_items = control[0];
    for(int i = blockIdx.x * kWarps + warp; i < short_items; i += gridDim.x * kWarps)
    {
        const int2 owner = owners[i];
        const int index = owner.x;
        const unsigned int v = (unsigned int)owner.y;
        const long long at = (long long)(index + 1 + lane) * chunk;
        const unsigned int other = __ballot_sync(0xffffffffu, !(at < tokens && sorted[at].x == v));
        const int parts = __ffs(other);                // the chunk itself and those up to the first that begins otherwise: at most kLongRun + 1
        for(int block = 0; block < blocks; block += 4)
        {
            T sum[4];
#pragma unroll
            for(int k = 0; k < 4; k++) sum[k] = P::zero();
#pragma unroll 2
            for(int j = 0; j < parts; j++)
            {
#pragma unroll
                for(int k = 0; k < 4; k++)
                {
                    const int column = ((block + k) * 32 + lane) * VEC;
                    if(column < E) sum[k] = P::add(sum[k], part(index, j, column));
                }
            }
#pragma unroll
            for(int k = 0; k < 4; k++)
            {
                const int column = ((block + k) * 32 + lane) * VEC;
                if(column < E) put_row<VEC>(dW + (long long)v * E + column, sum[k], scale, accumulate);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------

// Few positions and a small table: every CTA of the owner kernel reads all ids, and there is one for every 32 rows and 64 columns.
bool owners_do(int64_t tokens, int64_t E, int64_t V) { return tokens <= 2048 && E * V <= 3 << 20; }

// Positions of a chunk: enough chunks to fill the GPU, few enough that partial sums stay a small share of the traffic.
int chunk_of(int64_t tokens) { return tokens <= 32768 ? 16 : tokens <= 100000 ? 32 : 64; }

struct Layout { int64_t sorted, partial, owners, control, present, words; int chunks; };

Layout layout_of(int64_t tokens, int64_t E, int64_t V)
{
    auto up = [](int64_t words) { return (words + 3) / 4 * 4; };
    Layout l;
    l.chunks = (int)((tokens + chunk_of(tokens) - 1) / chunk_of(tokens));
    l.sorted = 0;
    l.partial = l.sorted + up(2 * tokens);
    l.owners = l.partial + up(2 * (int64_t)l.chunks * E);
    l.control = l.owners + up(2 * (int64_t)l.chunks);
    l.present = l.control + 4;
    l.words = l.present + up((V + 3) / 4);
    return l;
}

}  // namespace

}  // namespace onn

using namespace onn;

static bool sorted_sizes_ok(int64_t B, int64_t S, int64_t E, int64_t V)
{
    return B > 0 && S > 0 && E > 0 && V > 0 && E < (1LL << 23) && V < (1LL << 23) && B < (1LL << 31) && S < (1LL << 31) && B * S < (1LL << 31) - 65536;
}

extern "C" size_t onn_embedding_bwd_sorted_workspace_floats(int64_t B, int64_t S, int64_t E, int64_t V)
{
    if(!sorted_sizes_ok(B, S, E, V) || owners_do(B * S, E, V)) return 0;
    return (size_t)layout_of(B * S, E, V).words;
}

extern "C" int onn_embedding_bwd_sorted(const float* ids, const float* dY, const float* dY2, float* dW,
                                        int64_t B, int64_t S, int64_t E, int64_t V, int scale,
                                        float* workspace, uint32_t flags, void* stream)
{
    ONN_CHECK_ARG(ids && dY && dW && sorted_sizes_ok(B, S, E, V));
    ONN_CHECK_ARG((flags & ~ONN_ACCUMULATE) == 0);
    const int64_t tokens = B * S;
    const float scale_value = scale ? sqrtf((float)E) : 1.f;
    const int accumulate = (flags & ONN_ACCUMULATE) ? 1 : 0;
    cudaStream_t s = (cudaStream_t)stream;
    if(owners_do(tokens, E, V))
    {
        // a few CTAs for each SM if the table is that tall, but no more rows than fit in shared memory
        const int columns = (int)((E + kOwnerColumns - 1) / kOwnerColumns);
        int64_t owned = (V * columns + 2 * kSmCount - 1) / (2 * kSmCount);
        owned = owned < 1 ? 1 : owned > kMaxOwned ? kMaxOwned : owned;
        embedding_owner_kernel<<<dim3((unsigned)((V + owned - 1) / owned), columns), kOwnerThreads, 0, s>>>(
            ids, dY, dY2, dW, (int)tokens, (int)E, (int)V, scale_value, (int)owned, accumulate);
        count_launch();
        return launch_status();
    }
    if(!workspace) return ONN_ERR_WORKSPACE;
    ONN_CHECK_ARG(host_aligned16(workspace));
    const Layout l = layout_of(tokens, E, V);
    uint2* sorted = reinterpret_cast<uint2*>(workspace + l.sorted);
    float* partial = workspace + l.partial;
    int2* owners = reinterpret_cast<int2*>(workspace + l.owners);
    int* control = reinterpret_cast<int*>(workspace + l.control);
    unsigned char* present = reinterpret_cast<unsigned char*>(workspace + l.present);

    static PerDeviceBytes configured;
    if(!ensure_dynamic_smem(embedding_sort_kernel, configured, sizeof(SortShared))) return ONN_ERR_CUDA;
    int part_bits = 0;
    while((1 << part_bits) < kMinParts || (V >> part_bits) >= kMaxRows) part_bits++;
    embedding_sort_kernel<<<1u << part_bits, kSortThreads, sizeof(SortShared), s>>>(
        ids, sorted, control, present, (int)tokens, (int)V, part_bits);
    count_launch();
    if(launch_status() != ONN_OK) return ONN_ERR_CUDA;

    const bool vec = (E & 3) == 0 && host_aligned16(dY) && host_aligned16(dY2) && host_aligned16(dW);
    const int pieces = (int)(vec ? E / 4 : E);
    // threads of a chunk: the widest group that leaves fewest of its threads without a column
    int group = kReduceThreads;
    for(int g = kReduceThreads / 2; g >= 32; g /= 2)
        if((pieces + g - 1) / g * g < (pieces + group - 1) / group * group) group = g;
    const int chunk = chunk_of(tokens), groups = kReduceThreads / group;
    const int chunk_ctas = (l.chunks + groups - 1) / groups, zero_ctas = accumulate ? 0 : (int)((V + kZeroRows - 1) / kZeroRows);
    const int across = (pieces + group - 1) / group;
    const int64_t grid = (int64_t)chunk_ctas * across + zero_ctas;
    if(grid >= 1LL << 31) return ONN_ERR_LIMIT;
    auto add = [&](auto kernel)
    {
        return launch_overlapped(kernel, dim3((unsigned)grid), dim3(kReduceThreads), 0, s, (const uint2*)sorted,
                                 (const unsigned char*)present, dY, dY2, dW, partial, owners, control, (int)E, (int)V, chunk, l.chunks,
                                 chunk_ctas, across, group, scale_value, accumulate);
    };
    cudaError_t error = vec ? (dY2 ? add(embedding_chunk_kernel<4, true>) : add(embedding_chunk_kernel<4, false>))
                            : (dY2 ? add(embedding_chunk_kernel<1, true>) : add(embedding_chunk_kernel<1, false>));
    count_launch();
    if(error != cudaSuccess) return ONN_ERR_CUDA;
    auto join = [&](auto kernel)
    {
        return launch_overlapped(kernel, dim3(4 * kSmCount), dim3(kReduceThreads), 0, s, (const uint2*)sorted, (const float*)partial,
                                 (const int2*)owners, (const int*)control, dW, (int)E, chunk, l.chunks, scale_value, accumulate);
    };
    error = vec ? join(embedding_join_kernel<4>) : join(embedding_join_kernel<1>);
    count_launch();
    if(error != cudaSuccess) return ONN_ERR_CUDA;
    return launch_status();
}
