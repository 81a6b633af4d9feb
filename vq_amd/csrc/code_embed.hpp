// Tables of vectors that codes name: sums of their rows, and the gradient of the table.
//
// This translation unit must be compiled with -ffp-contract=off.
#pragma once
#include "code_rules.hpp"
#include "logprobs.hpp"

namespace vq {

// V values of a row from `s` on.  (Held in words: an array of 16-bit values is loaded one by one.)  A row's last piece, where it has no V values left,
// is read from V before its end on and written value by value; rows shorter than that have V = 1.
template <typename T, int V> struct Values {
    typedef typename T::Raw Raw;
    static constexpr int WORDS = V * (int)sizeof(Raw) / 4;
    struct __attribute__((packed, aligned(sizeof(Raw)))) Piece {
        uint32_t w[WORDS];
        __device__ __forceinline__ float at(int v) const {
            if constexpr (sizeof(Raw) == 4)
                return __uint_as_float(w[v]);
            else
                return T::up((Raw)(v & 1 ? w[v >> 1] >> 16 : w[v >> 1] & 0xffffu));
        }
    };
    static __device__ __forceinline__ Piece fetch(const Raw *s) { return *reinterpret_cast<const Piece *>(s); }
    // values from number `skip` on
    static __device__ __forceinline__ void store(Raw *to, const float (&x)[V], int skip = 0) {
        if (skip == 0) {
            Piece p;
#pragma unroll
            for (int q = 0; q < WORDS; ++q) {
                if constexpr (sizeof(Raw) == 4)
                    p.w[q] = __builtin_bit_cast(uint32_t, T::down(x[q]));
                else
                    p.w[q] = (uint32_t)T::down(x[2 * q]) | (uint32_t)T::down(x[2 * q + 1]) << 16;
            }
            *reinterpret_cast<Piece *>(to) = p;
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v >= skip) to[v] = T::down(x[v]);
        }
    }
};
template <typename T> struct Values<T, 1> {
    typedef typename T::Raw Raw;
    struct Piece {
        Raw value;
        __device__ __forceinline__ float at(int) const { return T::up(value); }
    };
    static __device__ __forceinline__ Piece fetch(const Raw *s) { return {*s}; }
    static __device__ __forceinline__ void store(Raw *to, const float (&x)[1], int = 0) { *to = T::down(x[0]); }
};
// Values of a lane: 16 bytes of the rows, or one where a row has fewer.
template <typename T> constexpr int wide() { return 16 / (int)sizeof(typename T::Raw); }

struct EmbedArgs {
    const void *table;
    int64_t ld;
    int k, dim, m;
    const void *codes;
    int code_bytes;
    int64_t n, code_stride;
    float scale;
    void *out;
    int64_t ld_out;
};

// out[i] = scale * sum over the stages s, in their order, of table[s * k + code].  The columns are cut into `slices` (of `pieces` vectors of 16 bytes of
// the table each): workgroup b has slice b % slices, so that with eight of them every XCD reads its own eighth of the tables' columns,
// which its L2 may hold.  1 << shift lanes of a row, rows side by side in a workgroup, a slice's further pieces by blockIdx.y.
// Where a row is the sum of many, what an XCD's L2 delivers and the additions count, two instructions per value, so that what else a row costs is kept
// small: offsets of 32 bits (Place) where a stage's table is below 4 GiB and its rows below 16 MiB apart, no conditions where all codes of a wave are
// codes.  65,536 x 8 stages of 1024 bf16, 51 us: 1.07 GB from L2 are 35 at the 30.7 TB/s that such reads reach alone, 27.6M vector instructions
// 27 (16.8M of them unpack and add, 17), 134 MB to memory 26.
template <typename T, typename O, int V, int NV, int BYTES, typename Place>
__global__ void __launch_bounds__(256) k_code_embed(EmbedArgs a, int shift, int slices, int pieces) {
    typedef typename T::Raw Raw;
    typedef Values<T, V> In;
    const int slice = blockIdx.x % (unsigned)slices;
    const int64_t row = (int64_t)(blockIdx.x / (unsigned)slices) * (256 >> shift) + (threadIdx.x >> shift);
    // NV pieces of a lane, as far apart as its row has lanes
    const int piece = (blockIdx.y * NV << shift) + (threadIdx.x & ((1 << shift) - 1)), end = min(pieces, (a.dim + V - 1) / V - slice * pieces);
    if (row >= a.n || piece >= end) return;
    const Place step = (Place)a.ld * (Place)sizeof(Raw), stage = (Place)a.k * step;
    const int64_t code0 = row * a.code_stride;
    float sum[NV][V];
    Place from[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        from[u] = (Place)min((slice * pieces + min(piece + (u << shift), end - 1)) * V, a.dim - V) * (Place)sizeof(Raw);
#pragma unroll
        for (int v = 0; v < V; ++v) sum[u][v] = 0.0f;
    }
    bool bad = false;
    const char *table = (const char *)a.table;  // of the stage
    const auto row_at = [&](uint32_t code) {
        if constexpr (sizeof(Place) == 4)
            return __umul24(code, step);  // (one instruction)
        else
            return (Place)code * step;
    };
    int s = 0;
    const auto stages = [&](auto count) {
        constexpr int S = decltype(count)::value;
        uint32_t code[S];  // (a negative one is above all others)
        bool fine = true;
#pragma unroll
        for (int j = 0; j < S; ++j) code[j] = (uint32_t)code_at(a.codes, BYTES, code0 + s + j);
#pragma unroll
        for (int j = 0; j < S; ++j) fine = fine && code[j] < (uint32_t)a.k;
        const auto fetch = [&](int j, int u) { return In::fetch(reinterpret_cast<const Raw *>(table + (int64_t)j * stage + (Place)(from[u] + row_at(code[j])))); };
        if (__ballot(!fine) == 0) {
            typename In::Piece p[S][NV];
#pragma unroll
            for (int j = 0; j < S; ++j)
#pragma unroll
                for (int u = 0; u < NV; ++u) p[j][u] = fetch(j, u);
#pragma unroll
            for (int j = 0; j < S; ++j)
#pragma unroll
                for (int u = 0; u < NV; ++u)
#pragma unroll
                    for (int v = 0; v < V; ++v) sum[u][v] += p[j][u].at(v);
        } else {
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (code[j] < (uint32_t)a.k) {
#pragma unroll
                    for (int u = 0; u < NV; ++u) {
                        const typename In::Piece p = fetch(j, u);
#pragma unroll
                        for (int v = 0; v < V; ++v) sum[u][v] += p.at(v);
                    }
                } else if ((int32_t)code[j] >= 0)
                    bad = true;
        }
        s += S;
        table += (int64_t)S * stage;
    };
    while (s + 8 <= a.m) stages(std::integral_constant<int, 8>());
    if (a.m & 4) stages(std::integral_constant<int, 4>());
    if (a.m & 2) stages(std::integral_constant<int, 2>());
    if (a.m & 1) stages(std::integral_constant<int, 1>());
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        if (u > 0 && piece + (u << shift) >= end) break;
        const int place = (slice * pieces + piece + (u << shift)) * V, at = min(place, a.dim - V);
#pragma unroll
        for (int v = 0; v < V; ++v) sum[u][v] = bad ? __builtin_nanf("") : a.scale * sum[u][v];
        Values<O, V>::store((typename O::Raw *)a.out + row * a.ld_out + at, sum[u], place - at);
    }
}

// ---- the positions by code ---------------------------------------------------------------------------
struct ListArgs {
    const void *codes;
    int64_t code_stride;
    int n, k, width;  // codes of a bucket
    int share, shares;  // positions of a share of the list, and how many there are
    int32_t *start, *rows, *edges;  // edges: the code of each kLongCode-th position of the list
    int32_t *counts, *below;  // of several shares: [stage][share][code], [stage][share][bucket]
};

// A workgroup has a bucket of codes (blockIdx.x), a share of the positions (blockIdx.y) and a stage (blockIdx.z); it reads all codes of its
// share, counts those below its bucket, whose number is where its part of the list begins, and those in it, by wave and code.  Each wave has a
// run of the positions, so that the order within a code is that of the positions; the few of them that its bucket has it keeps in LDS, and
// reads its run again only where they are more than fit there.  With one share the workgroup goes on and writes its part of the list; of several
// shares the counts are added up first, by the launch after (PLACE).
constexpr int kQueue = kListQueue;
template <int WAVES, int BYTES, bool COUNT, bool PLACE>
__global__ void __launch_bounds__(64 * WAVES) k_code_lists(ListArgs a) {
    extern __shared__ int hist[];  // [wave][code of the bucket], and (PLACE) [wave][kQueue]
    __shared__ int below_of[WAVES], total_of[WAVES], sums_of[COUNT ? 1 : 2][COUNT ? 1 : 64 * WAVES];
    static_assert(COUNT || sizeof(below_of) + sizeof(total_of) + sizeof(sums_of) == kListBeside, "as the plan counts it");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), stage = blockIdx.z, share = blockIdx.y, buckets = gridDim.x;
    const int lo = blockIdx.x * a.width, width = min(a.width, a.k - lo);
    const int first = (int)min((int64_t)a.n, (int64_t)share * a.share), end = (int)min((int64_t)a.n, (int64_t)first + a.share);
    const int run = ((end - first) + 64 * WAVES - 1) / (64 * WAVES) * 64, from = min(end, first + wave * run), to = min(end, from + run);
    int *mine = hist + wave * a.width;
    uint2 *queue = reinterpret_cast<uint2 *>(hist + ((WAVES * a.width + 1) & ~1)) + wave * kQueue;
    for (int i = tid; i < WAVES * a.width; i += 64 * WAVES) hist[i] = 0;
    __syncthreads();
    constexpr int AHEAD = 16;
    const auto code_of = [&](int i) { return i < to ? (uint32_t)code_at(a.codes, BYTES, (int64_t)i * a.code_stride + stage) : 0xffffffffu; };
    int below = 0, queued = 0;
    for (int i = from + lane; i - lane < to; i += 64 * AHEAD) {
        uint32_t c[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) c[j] = code_of(i + 64 * j);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            below += c[j] < (uint32_t)lo;
            const uint32_t code = c[j] - (uint32_t)lo;
            const unsigned long long who = __ballot(code < (uint32_t)width);
            if (!who) continue;  // uniform
            const int place = queued + __popcll(who & ((1ull << lane) - 1));
            if (code < (uint32_t)width) {
                atomicAdd(&mine[code], 1);
                if (PLACE && place < kQueue) queue[place] = make_uint2(code, i + 64 * j);
            }
            queued += __popcll(who);
        }
    }
    below = (int)over_group<64>((uint32_t)below, 0u, [](uint32_t x, uint32_t y) { return x + y; });
    if (lane == 0) below_of[wave] = below;
    __syncthreads();
    int32_t *counts = a.counts + (int64_t)stage * a.shares * a.k, *belows = a.below + (int64_t)stage * a.shares * buckets;
    if constexpr (!PLACE) {
        for (int i = tid; i < width; i += 64 * WAVES) {
            int sum = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) sum += hist[w * a.width + i];
            counts[(int64_t)share * a.k + lo + i] = sum;
        }
        if (tid == 0) {
            int sum = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) sum += below_of[w];
            belows[share * buckets + blockIdx.x] = sum;
        }
        return;
    }
    int base = 0;
    if constexpr (COUNT) {
#pragma unroll
        for (int w = 0; w < WAVES; ++w) base += below_of[w];
    } else {
        for (int s = tid; s < a.shares; s += 64 * WAVES) base += belows[s * buckets + blockIdx.x];
        base = (int)over_group<64>((uint32_t)base, 0u, [](uint32_t x, uint32_t y) { return x + y; });
        if (lane == 0) total_of[wave] = base;
        __syncthreads();
        base = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) base += total_of[w];
        __syncthreads();
    }
    // where each code's list begins, in it this share's part, and in that each wave's; a lane per code, and as many lanes more as there are
    // for the counts of the shares
    int32_t *start = a.start + (int64_t)stage * (a.k + 1);
    int all = 0, ahead = 0;  // of code tid: positions in all shares, in the shares before this one
    if constexpr (COUNT) {
        if (tid < width) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w) all += hist[w * a.width + tid];
        }
    } else {
        const int sides = 64 * WAVES / width, side = tid / width, c = tid - side * width;
        if (side < sides) {
            for (int s = side; s < a.shares; s += 16 * sides) {
                int here[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) here[j] = s + j * sides < a.shares ? counts[(int64_t)(s + j * sides) * a.k + lo + c] : 0;
#pragma unroll
                for (int j = 0; j < 16; ++j) all += here[j], ahead += s + j * sides < share ? here[j] : 0;
            }
        }
        sums_of[0][tid] = all;
        sums_of[1][tid] = ahead;
        __syncthreads();
        if (tid < width) {
            for (int o = 1; o < sides; ++o) all += sums_of[0][o * width + tid], ahead += sums_of[1][o * width + tid];
        } else
            all = 0;
    }
    int upto = all;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 63) total_of[wave] = upto;
    __syncthreads();
    int at = base + upto - all;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) at += w < wave ? total_of[w] : 0;
    if (tid < width) {
        if (share == 0) {
            start[lo + tid] = at;
            if (lo + tid == a.k - 1) start[a.k] = at + all;
        }
        at += ahead;
        int here[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) here[w] = hist[w * a.width + tid];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            hist[w * a.width + tid] = at;
            at += here[w];
        }
    }
    __syncthreads();
    int32_t *rows = a.rows + (int64_t)stage * a.n, *edges = a.edges + (int64_t)stage * embed_edges(a.n);
    // up to 64 positions in their order, those with `own` in the bucket
    const auto put = [&](bool own, uint32_t code, int position) {
        // the lanes with the same code: bit by bit of it
        unsigned long long same = __ballot(own);
        for (int bit = 1; bit < a.width; bit <<= 1) {
            const unsigned long long set = __ballot((code & bit) != 0);
            same &= code & bit ? set : ~set;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int place = own ? mine[code] + rank : 0;
        wave_sync();
        if (own && rank == 0) mine[code] = place + __popcll(same);
        wave_sync();
        if (own) {
            rows[place] = position;
            if (place % kLongCode == 0) edges[place / kLongCode] = lo + (int)code;
        }
    };
    if (queued <= kQueue) {  // uniform
        for (int i = lane; i - lane < queued; i += 64) {
            const uint2 o = queue[min(i, queued - 1)];
            put(i < queued, o.x, (int)o.y);
        }
    } else {
        for (int i = from + lane; i - lane < to; i += 64 * AHEAD) {
            uint32_t c[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) c[j] = code_of(i + 64 * j) - (uint32_t)lo;
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (__ballot(c[j] < (uint32_t)width)) put(c[j] < (uint32_t)width, c[j], i + 64 * j);
        }
    }
}

// ---- the sums ------------------------------------------------------------------------------------------
struct SumArgs {
    const void *g;
    int64_t ld;
    int n, dim, k;
    float scale;
    int accumulate;
    void *grad;
    int64_t ld_grad;
    const void *few_codes;  // (where the workgroups make their own lists)
    int code_bytes;
    int64_t code_stride;
    const int32_t *start, *rows, *edges;
    float *partial;  // [stage][chunk][2][padded dim]
    int chunks, padded, codes, groups, across, first;  // codes of a workgroup; workgroups of codes; of columns, and the first of these
};

constexpr int kGroupCodes = 128;  // codes of a workgroup at most
// A code of more positions than this is summed by the whole workgroup.  (Where a workgroup has few codes it sums one alone sooner than a group of
// lanes sums 32 rows.)  16,384 x 1280 bf16 of 65,536 uneven codes 96 us, with 16 instead of 32 members 115; 100,000 x 128 of 1024 uneven codes 35, with 64 78;
// 1000 x 100 of 50 codes in one launch 12.9, with 5 instead of 10 15.6, with 20 12.8.
// kOwnMost: no group of lanes sums more, however many such codes a workgroup has, so that no sum is of more than 76 roundings behind one another
// (uncapped 1024 and more; the cap and eights: 100,000 x 64 bf16 of 1000 uneven codes 32.4 -> 28.6 us).
constexpr int kOwnMembers = 32, kFewMembers = 10, kOwnMost = 512;

// Adds V columns of the members number a, a + step, ... below b of a list, in that order, eight at a time whose sum is added: a rounding for each of
// 512 members behind one another would lose nine of the 24 bits.
template <typename T, int V, typename Rows>
__device__ __forceinline__ void sum_members(const SumArgs &s, Rows rows, int a, int b, int step, int at, float (&sum)[V]) {
    typedef typename T::Raw Raw;
    typedef Values<T, V> In;
    constexpr int AHEAD = 8;
    const Raw *g = (const Raw *)s.g + at;
    for (int p = a; p < b; p += AHEAD * step) {
        // (behind the last member the last one again, which is not added: loads under a condition would wait for one another)
        int row[AHEAD];
        typename In::Piece x[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) row[j] = rows[min(p + j * step, b - 1)];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) x[j] = In::fetch(g + (int64_t)row[j] * s.ld);
        if (p + (AHEAD - 1) * step < b) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                sum[v] += ((x[0].at(v) + x[1].at(v)) + (x[2].at(v) + x[3].at(v))) + ((x[4].at(v) + x[5].at(v)) + (x[6].at(v) + x[7].at(v)));
        } else {
#pragma unroll
            for (int j = 0; j < AHEAD - 1; ++j)
                if (p + j * step < b) {
#pragma unroll
                    for (int v = 0; v < V; ++v) sum[v] += x[j].at(v);
                }
        }
    }
}

// Rows without members, most of a large table's, of 64 codes and up to 16 KB of their columns: whole lines that pass the caches.  These
// workgroups come last: zeros written beside the reads of the sums made both slower (16,384 x 1280 bf16 to 65,536 f32 rows 101 us, apart
// 77).
constexpr int kZeroCodes = 64, kZeroBytes = 16384;
template <typename O, int VO> __device__ __forceinline__ void zero_piece(typename O::Raw *to, int c, int end) {  // [c, c + VO) below end
    const float zeros[VO] = {};
    if (c + VO <= end) {
        Values<O, VO>::store(to + c, zeros);
    } else {
#pragma unroll
        for (int v = 0; v < VO; ++v)
            if (c + v < end) to[c + v] = O::down(0.0f);
    }
}
template <typename O> __device__ __forceinline__ void write_zeros(const SumArgs &a, unsigned id, int stage, int *list, int *count) {
    typedef typename O::Raw Out;
    constexpr int VO = wide<O>(), PIECE = kZeroBytes / (int)sizeof(Out);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned pieces = (unsigned)(a.dim + PIECE - 1) / PIECE;
    const int64_t code = (int64_t)(id / pieces) * kZeroCodes + tid;
    const int column = (int)(id % pieces) * PIECE, end = min(a.dim, column + PIECE);
    const int32_t *start = a.start + (int64_t)stage * (a.k + 1);
    if (wave == 0) {
        const bool empty = code < a.k && start[code] == start[code + 1];
        const unsigned long long who = __ballot(empty);
        if (empty) list[__popcll(who & ((1ull << lane) - 1))] = (int)code;
        if (lane == 0) *count = __popcll(who);
    }
    __syncthreads();
    const bool past = ((uintptr_t)a.grad & 15) == 0 && a.ld_grad % VO == 0 && a.dim % VO == 0;  // whole pieces of 16 aligned bytes
    // 1 << shift lanes of a row, so that rows of a few bytes lie side by side in a wave
    int shift = 0;
    while (shift < 6 && VO << shift < end - column) ++shift;
    for (int i = tid >> shift; i < *count; i += 256 >> shift) {
        Out *to = (Out *)a.grad + ((int64_t)stage * a.k + list[i]) * a.ld_grad;
        for (int c = column + (tid & ((1 << shift) - 1)) * VO; c < end; c += VO << shift) {
            if (past) {
                typedef uint32_t Four __attribute__((ext_vector_type(4)));
                __builtin_nontemporal_store(Four{0, 0, 0, 0}, reinterpret_cast<Four *>(to + c));
            } else {
                zero_piece<O, VO>(to, c, end);
            }
        }
    }
}

// Rows of the gradient: 16 lanes sum V columns each of a code's members.  The first a.groups workgroups take codes, those behind them the
// chunks of the list that belong to codes of more than kLongCode members; a.across workgroups side by side have the columns,
// 16 * V each; the last ones write the rows without members.  blockIdx.z: stages.
// FEW: up to kFewPositions of them, which every workgroup lists for its own codes: one launch instead of two.
// Five waves to a SIMD, which 96 registers allow; sums of 16-bit rows to f32, which would spill, four (FEW spills three registers for them).
template <typename T, typename O, int V, bool FEW>
__global__ void __launch_bounds__(256, FEW || sizeof(typename T::Raw) == 4 || sizeof(typename O::Raw) == 2 ? 5 : 4) k_embed_sums(SumArgs a) {
    typedef typename T::Raw Raw;
    typedef typename O::Raw Out;
    constexpr int COLUMNS = 16 * V, VO = V == 1 ? 1 : wide<O>();
    __shared__ float red[16][COLUMNS];
    __shared__ int begin[kGroupCodes], behind[kGroupCodes], count[4];
    __shared__ uint8_t which[3][kGroupCodes];
    __shared__ int few[FEW ? kFewPositions : 1], queue[FEW ? kFewPositions + 8 : 1], queued[4];
    const int tid = threadIdx.x, sub = tid >> 4, column = (a.first + blockIdx.x % (unsigned)a.across) * COLUMNS, place = column + (tid & 15) * V, at = min(place, a.dim - V), stage = blockIdx.z;
    const bool used = place < a.dim;  // this lane has columns
    if (!FEW && blockIdx.x >= (unsigned)(a.groups + a.chunks) * (unsigned)a.across) {
        write_zeros<O>(a, blockIdx.x - (unsigned)(a.groups + a.chunks) * (unsigned)a.across, stage, begin, &count[0]);
        return;
    }
    const int group = blockIdx.x / (unsigned)a.across;
    const int32_t *start = a.start + (int64_t)stage * (a.k + 1), *rows = a.rows + (int64_t)stage * a.n;
    const auto list = [&] {
        if constexpr (FEW)
            return (const int *)few;
        else
            return rows;
    }();
    Out *grad = (Out *)a.grad + (int64_t)stage * a.k * a.ld_grad;
    float sum[V];
    // a lane's sums to their columns' places (the last piece of a row reaches back over columns of another)
    const auto lay_out = [&] {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (at + v >= column) red[sub][at - column + v] = sum[v];
    };
    // results: scaled, added to what is there
    const auto put = [&](Out *to, float (&y)[VO], int skip) {
        if (a.accumulate) {
            const typename Values<O, VO>::Piece old = Values<O, VO>::fetch(to);
#pragma unroll
            for (int v = 0; v < VO; ++v) y[v] = __builtin_fmaf(a.scale, y[v], old.at(v));
        } else {
#pragma unroll
            for (int v = 0; v < VO; ++v) y[v] *= a.scale;
        }
        Values<O, VO>::store(to, y, skip);
    };
    const auto put_one = [&](Out *to, float y) { *to = O::down(a.accumulate ? __builtin_fmaf(a.scale, y, O::up(*to)) : a.scale * y); };
    // all 16 groups of lanes sum members [from, to); the sums of COLUMNS columns are in the first lanes then
    const auto together = [&](int from, int to) {
        if (used) {
#pragma unroll
            for (int v = 0; v < V; ++v) sum[v] = 0.0f;
            sum_members<T, V>(a, list, from + sub, to, 16, at, sum);
            lay_out();
        }
        __syncthreads();
        float total = 0.0f;
        if (tid < COLUMNS && column + tid < a.dim) {
#pragma unroll
            for (int j = 0; j < 16; ++j) total += red[j][tid];
        }
        __syncthreads();
        return total;
    };
    if (!FEW && group >= a.groups) {
        const int chunk = group - a.groups, all = start[a.k], first = chunk * kLongCode, last = min(all, first + kLongCode) - 1;
        if (first > last) return;
        // the codes of the chunk's first position and, where another one's list goes on behind the chunk, of that (no other list that
        // begins in the chunk is long)
        const int32_t *edges = a.edges + (int64_t)stage * embed_edges(a.n);
        const int c0 = edges[chunk], then = last + 1 < all ? edges[chunk + 1] : c0, c1 = start[then] <= last ? then : c0;
        for (int slot = 0; slot < 2; ++slot) {
            const int c = slot ? c1 : c0;
            if (slot && c1 == c0) break;
            const int s0 = start[c], s1 = start[c + 1];
            if (s1 - s0 <= kLongCode) continue;
            const float total = together(max(s0, first), min(s1, last + 1));
            if (tid < COLUMNS && column + tid < a.dim) a.partial[(((int64_t)stage * a.chunks + chunk) * 2 + slot) * a.padded + column + tid] = total;
        }
        return;
    }
    // the workgroup's codes by the number of their members: a group of lanes each, or the whole workgroup
    const int64_t from = (int64_t)group * a.codes;
    if (tid < 4) count[tid] = 0;
    int s0 = 0, s1 = 0;
    if constexpr (FEW) {
        // the positions of these codes, in their order, by wave; then each code's, a lane per code
        const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        uint32_t code[kFewPositions / 256];
#pragma unroll
        for (int j = 0; j < kFewPositions / 256; ++j) {
            const int i = wave * (kFewPositions / 4) + j * 64 + lane;
            code[j] = i < a.n ? (uint32_t)(code_at(a.few_codes, a.code_bytes, (int64_t)i * a.code_stride + stage) - from) : 0xffffffffu;
        }
        const uint32_t codes = (uint32_t)min((int64_t)a.codes, a.k - from);
        unsigned long long who[kFewPositions / 256];
        int found = 0;
#pragma unroll
        for (int j = 0; j < kFewPositions / 256; ++j) {
            who[j] = __ballot(code[j] < codes);
            found += __popcll(who[j]);
        }
        if (lane == 0) queued[wave] = found;
        __syncthreads();
        int at = 0, total = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            at += w < wave ? queued[w] : 0;
            total += queued[w];
        }
#pragma unroll
        for (int j = 0; j < kFewPositions / 256; ++j) {
            if (code[j] < codes) queue[at + __popcll(who[j] & ((1ull << lane) - 1))] = (wave * (kFewPositions / 4) + j * 64 + lane) * kGroupCodes + (int)code[j];
            at += __popcll(who[j]);
        }
        if (tid < 8) queue[total + tid] = -1;  // up to a whole eight: none of these codes (there are fewer than kGroupCodes)
        __syncthreads();
        if (tid < kFewCodes) {
            int members = 0;
            for (int i = 0; i < total; i += 8) {
                int o[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) o[u] = queue[i + u];
#pragma unroll
                for (int u = 0; u < 8; ++u) members += (o[u] & (kGroupCodes - 1)) == tid;
            }
            int upto = members;
#pragma unroll
            for (int d = 1; d < kFewCodes; d <<= 1) {
                const int o = __shfl_up(upto, d);
                if (lane >= d) upto += o;
            }
            s0 = upto - members;
            s1 = s0;
            for (int i = 0; i < total; i += 8) {
                int o[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) o[u] = queue[i + u];
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if ((o[u] & (kGroupCodes - 1)) == tid) few[s1++] = o[u] / kGroupCodes;
            }
        }
    } else if (tid < a.codes && from + tid < a.k) {
        s0 = start[from + tid];
        s1 = start[from + tid + 1];
    }
    __syncthreads();
    const bool has = tid < a.codes && from + tid < a.k;
    const int members = s1 - s0;
    if (has && members > (FEW ? kFewMembers : kOwnMembers) && members <= kLongCode) atomicAdd(&count[3], 1);
    __syncthreads();
    if (has) {
        // (16 codes side by side take the time of the longest, each by all lanes that of their sum: the more there are, the longer they may be)
        const int own = min(kOwnMost, (FEW ? kFewMembers : kOwnMembers) * max(1, count[3]));
        begin[tid] = s0;
        behind[tid] = s1;
        if (members <= kLongCode) {
            const int kind = members == 0 ? 2 : members <= own ? 0 : 1;
            which[kind][atomicAdd(&count[kind], 1)] = (uint8_t)tid;  // (in whatever order: each is a sum of its own)
        }
    }
    __syncthreads();
    // codes of few members, a group of lanes each: the first two members of four codes at a time, since most have no more
    constexpr int SIDE = 4, EARLY = 2;
    for (int i = sub; i < count[0]; i += 16 * SIDE) {  // (lanes without columns of the row go along)
        typename Values<T, V>::Piece x[SIDE][EARLY];
        int row[SIDE][EARLY];
#pragma unroll
        for (int u = 0; u < SIDE; ++u) {  // (beyond the last code or member the last one again)
            const int j = which[0][min(i + 16 * u, count[0] - 1)], s0 = begin[j], s1 = behind[j];
#pragma unroll
            for (int e = 0; e < EARLY; ++e) row[u][e] = list[min(s0 + e, s1 - 1)];
        }
#pragma unroll
        for (int u = 0; u < SIDE; ++u)
#pragma unroll
            for (int e = 0; e < EARLY; ++e) x[u][e] = Values<T, V>::fetch((const Raw *)a.g + at + (int64_t)row[u][e] * a.ld);
#pragma unroll
        for (int u = 0; u < SIDE; ++u) {
            if (i + 16 * u >= count[0]) break;
            const int j = which[0][i + 16 * u], s0 = begin[j], s1 = behind[j];
#pragma unroll
            for (int v = 0; v < V; ++v) sum[v] = x[u][0].at(v);
            if (s0 + 1 < s1) {
#pragma unroll
                for (int v = 0; v < V; ++v) sum[v] += x[u][1].at(v);
            }
            if (s0 + EARLY < s1) sum_members<T, V>(a, list, s0 + EARLY, s1, 1, at, sum);
            Out *to = grad + (from + j) * a.ld_grad;
            if constexpr (VO == V) {
                if (used) put(to + at, sum, place - at);
            } else {  // the lanes' 16 bytes of results side by side
                wave_sync();
                if (used) lay_out();
                wave_sync();
#pragma unroll
                for (int c = 0; c < COLUMNS; c += 16 * VO) {
                    const int col = c + (tid & 15) * VO, rest = a.dim - column - col;
                    float y[VO];
                    if (col < COLUMNS && rest > 0) {
#pragma unroll
                        for (int v = 0; v < VO; ++v) y[v] = red[sub][col + v];
                        if (rest >= VO) {
                            put(to + column + col, y, 0);
                        } else {
#pragma unroll
                            for (int v = 0; v < VO; ++v)
                                if (v < rest) put_one(to + column + col + v, y[v]);
                        }
                    }
                }
            }
        }
    }
    __syncthreads();
    const int n_longer = count[1];
    for (int i = 0; i < n_longer; ++i) {
        const int j = which[1][i];
        const float total = together(begin[j], behind[j]);
        if (tid < COLUMNS && column + tid < a.dim) put_one(grad + (from + j) * a.ld_grad + column + tid, total);
    }
    if (FEW && !a.accumulate) {
        for (int i = sub; i < count[2]; i += 16) {
            Out *to = grad + (from + which[2][i]) * a.ld_grad;
            for (int c = column + (tid & 15) * VO; c < min(a.dim, column + COLUMNS); c += 16 * VO) zero_piece<O, VO>(to, c, min(a.dim, column + COLUMNS));
        }
    }
}

// The sums of the chunks of a code of more than kLongCode members, by the workgroup of the chunk in which the code's list begins:
// 64 columns (blockIdx.y), 16 groups of 16 lanes that share the chunks, a million of them where all positions have one code: summed in 64 bits.
template <typename O>
__global__ void __launch_bounds__(256) k_embed_join(SumArgs a) {
    typedef typename O::Raw Out;
    __shared__ double red[16][64];
    const int tid = threadIdx.x, sub = tid >> 4, column = blockIdx.y * 64, at = column + (tid & 15) * 4, stage = blockIdx.z, chunk = blockIdx.x;
    const int32_t *start = a.start + (int64_t)stage * (a.k + 1), *edges = a.edges + (int64_t)stage * embed_edges(a.n);
    const int all = start[a.k], first = chunk * kLongCode, last = first + kLongCode - 1;
    if (last + 1 >= all) return;  // (a long list that begins in a chunk goes on behind it)
    const int code = edges[chunk + 1], s0 = start[code], s1 = start[code + 1];
    if (s1 - s0 <= kLongCode || s0 < first || s0 > last) return;
    const int end = (s1 - 1) / kLongCode;  // the last chunk with members of this code
    const float *partial = a.partial + (int64_t)stage * a.chunks * 2 * a.padded;
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    if (at < a.dim) {
        for (int c = chunk + sub; c <= end; c += 16) {
            const int slot = c == chunk && s0 != first ? 1 : 0;
            const float4 x = *reinterpret_cast<const float4 *>(partial + ((int64_t)c * 2 + slot) * a.padded + at);
            sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w;
        }
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) red[sub][(tid & 15) * 4 + v] = sum[v];
    __syncthreads();
    if (tid >= 64 || column + tid >= a.dim) return;
    double all_of = 0.0;
#pragma unroll
    for (int j = 0; j < 16; ++j) all_of += red[j][tid];
    const float total = (float)all_of;
    Out *to = (Out *)a.grad + ((int64_t)stage * a.k + code) * a.ld_grad + column + tid;
    *to = O::down(a.accumulate ? __builtin_fmaf(a.scale, total, O::up(*to)) : a.scale * total);
}

}  // namespace vq
