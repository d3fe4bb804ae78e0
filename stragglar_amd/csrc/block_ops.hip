// Block operators of an emulated group: what its ranks exchange inside a model's block.
//
//   sar_route             slots (token, choice) sorted by expert, stable
//   sar_dispatch          tokens to their rows in expert order (and the gradient of sar_combine's rows)
//   sar_combine           a token's rows back as their weighted sum (and the gradient of sar_dispatch)
//   sar_reduce_norm       sum over the ranks' partial outputs, norm, gate, residual, norm, a copy for every rank
//
// All of it is bound by HBM, so the kernels read every input once and keep what they need again in registers.  Rows
// are moved as 16-byte vectors whatever their alignment: gfx950 takes 16-byte accesses at any element boundary, and a
// row whose length is no whole number of vectors ends in a vector that overlaps the one before it (both lanes compute
// and store the same bits; sums leave the doubled elements out).  Only rows shorter than one vector go element by
// element.
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

#include "errors.hpp"
#include "sar.h"

namespace sar {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef u4 u4_any __attribute__((aligned(2)));   // 16 bytes at any element boundary
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));

constexpr int kWave = 64;

// ---- vectors of elements ------------------------------------------------------------------------------------
// VE elements of a type: 16 bytes of them, or one where rows are shorter than that.
template <int DT> struct ElemSize { static constexpr int value = DT == SAR_F32 ? 4 : 2; };
template <int DT> constexpr int kVec = 16 / ElemSize<DT>::value;

template <int DT, int VE> struct Raw { typedef u4 T; };
template <> struct Raw<SAR_F32, 1> { typedef uint32_t T; };
template <> struct Raw<SAR_F16, 1> { typedef uint16_t T; };
template <> struct Raw<SAR_BF16, 1> { typedef uint16_t T; };

// NT: streaming, for what nobody reads again soon.
template <int DT, int VE, bool NT = false>
__device__ __forceinline__ typename Raw<DT, VE>::T load(const char* base, uint32_t byte) {
    if constexpr (VE == 1) {
        typedef __attribute__((address_space(1))) const typename Raw<DT, VE>::T* P;
        return *(P)(base + byte);
    } else {
        typedef __attribute__((address_space(1))) const u4_any* P;
        return NT ? (u4)__builtin_nontemporal_load((P)(base + byte)) : (u4)*(P)(base + byte);
    }
}
template <int DT, int VE, bool NT = false>
__device__ __forceinline__ void store(char* base, uint32_t byte, typename Raw<DT, VE>::T v) {
    if constexpr (VE == 1) {
        typedef __attribute__((address_space(1))) typename Raw<DT, VE>::T* P;
        *(P)(base + byte) = v;
    } else {
        typedef __attribute__((address_space(1))) u4_any* P;
        if (NT) __builtin_nontemporal_store((u4_any)v, (P)(base + byte));
        else *(P)(base + byte) = v;
    }
}

// Where a lane's vector `vec` of a row lies.  Behind the row's end it is the last vector again: loads need no branch (a
// load behind a branch is waited for before the next is issued), sums leave out the first `skip` elements (doubled
// ones, or all), stores ask `in`.
template <int DT, int VE>
struct Place {
    uint32_t elem, skip;
    bool in;
    __device__ __forceinline__ Place(uint32_t vec, uint32_t nvec, uint32_t dim) {
        elem = min(vec * VE, dim - VE);
        skip = vec * VE - elem;
        in = vec < nvec;
    }
    __device__ __forceinline__ uint32_t byte() const { return elem * (uint32_t)ElemSize<DT>::value; }
};

// Loads `count` rows' vectors in batches as large as they come and hands each to `use` in order: all loads of a batch
// are on their way before the first is waited for.
template <int N, class Load, class Use>
__device__ __forceinline__ void batch(uint32_t first, Load&& ld, Use&& use) {
    decltype(ld(0u)) v[N];
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] = ld(first + q);
#pragma unroll
    for (int q = 0; q < N; ++q) use(v[q]);
}
template <int MOST, class Load, class Use>
__device__ __forceinline__ void in_batches(uint32_t count, Load&& ld, Use&& use) {
    uint32_t s = 0;
    for (; s + MOST <= count; s += MOST) batch<MOST>(s, ld, use);
    if constexpr (MOST > 4) if (s + 4 <= count) { batch<4>(s, ld, use); s += 4; }
    if constexpr (MOST > 2) if (s + 2 <= count) { batch<2>(s, ld, use); s += 2; }
    if constexpr (MOST > 1) if (s < count) batch<1>(s, ld, use);
}

__device__ __forceinline__ float widen(uint32_t bits, int dt) {   // one 16-bit element in the low half
    if (dt == SAR_BF16) return __uint_as_float(bits << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

template <int DT, int VE>
__device__ __forceinline__ void unpack(typename Raw<DT, VE>::T r, float* x) {
    if constexpr (VE == 1) {
        if constexpr (DT == SAR_F32) x[0] = __uint_as_float(r);
        else x[0] = widen(r, DT);
    } else if constexpr (DT == SAR_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
    } else if constexpr (DT == SAR_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(r[i] << 16);
            x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t bits = r[i];   // a value of its own: __builtin_bit_cast of a vector's element reads element 0
            const h2 h = __builtin_bit_cast(h2, bits);
            x[2 * i] = (float)h.x;
            x[2 * i + 1] = (float)h.y;
        }
    }
}

// The one rounding of a result: to nearest, ties to even.
template <int DT, int VE>
__device__ __forceinline__ typename Raw<DT, VE>::T pack(const float* x) {
    if constexpr (VE == 1) {
        if constexpr (DT == SAR_F32) return __float_as_uint(x[0]);
        else if constexpr (DT == SAR_F16) return __builtin_bit_cast(uint16_t, (_Float16)x[0]);
        else return __builtin_bit_cast(uint16_t, (__bf16)x[0]);
    } else {
        u4 r;
        if constexpr (DT == SAR_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f2 p;
                p.x = x[2 * i];
                p.y = x[2 * i + 1];
                if constexpr (DT == SAR_BF16) r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf2));
                else r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, h2));
            }
        }
        return r;
    }
}

// VE parameters (weights, gate) from element `elem` on, held in DT or in 32 bits.
template <int DT, int VE>
__device__ __forceinline__ void load_param(const char* p, bool f32, uint32_t elem, float* x) {
    if (DT == SAR_F32 || f32) {
        if constexpr (VE == 1) {
            x[0] = __uint_as_float(load<SAR_F32, 1>(p, elem * 4u));
        } else {
#pragma unroll
            for (int q = 0; q < VE / 4; ++q) unpack<SAR_F32, 4>(load<SAR_F32, 4>(p, elem * 4u + 16u * q), x + 4 * q);
        }
    } else {
        unpack<DT, VE>(load<DT, VE>(p, elem * (uint32_t)ElemSize<DT>::value), x);
    }
}
template <int DT>
__device__ __forceinline__ float load_one(const char* p, bool f32, uint64_t elem) {
    float x;
    if (DT == SAR_F32 || f32) x = ((const float*)p)[elem];
    else unpack<DT, 1>(load<DT, 1>(p + elem * (uint64_t)ElemSize<DT>::value, 0), &x);
    return x;
}
template <int DT>
__device__ __forceinline__ void store_one(char* p, bool f32, uint64_t elem, float x) {
    if (DT == SAR_F32 || f32) ((float*)p)[elem] = x;
    else store<DT, 1>(p + elem * (uint64_t)ElemSize<DT>::value, 0, pack<DT, 1>(&x));
}

// ---- sums over lanes ----------------------------------------------------------------------------------------
// The sum over a wave, in every lane; always the same order (lanes to the right, then rows of 16, then halves).
__device__ __forceinline__ float wave_sum(float x) {
#define SAR_DPP_ADD(ctrl, rows) \
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, rows, 0xf, false))
    SAR_DPP_ADD(0x111, 0xf);   // from 1, 2, 4, 8 lanes to the left within a row of 16
    SAR_DPP_ADD(0x112, 0xf);
    SAR_DPP_ADD(0x114, 0xf);
    SAR_DPP_ADD(0x118, 0xf);
    SAR_DPP_ADD(0x142, 0xa);   // last lane of rows 0 and 2 to rows 1 and 3
    SAR_DPP_ADD(0x143, 0xc);   // lane 31 to the upper half
#undef SAR_DPP_ADD
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), kWave - 1));
}

// Sums over the waves that share a row (all of the workgroup's, or `waves` consecutive ones of it), in every lane.
// `turn` alternates between two halves of the scratch, so that one barrier a sum is enough: a half is written again only
// after everybody has passed the barrier of the sum in between.  The whole workgroup takes part in every sum.
struct RowSum {
    float* scratch;   // 2 * 2 * 16 floats of LDS
    uint32_t turn, waves, wave, lane;
    __device__ __forceinline__ void operator()(float& a, float& b) {
        a = wave_sum(a);
        b = wave_sum(b);
        if (waves == 1) return;
        float* s = scratch + 32u * (turn & 1u);
        ++turn;
        if (lane == 0) { s[wave] = a; s[16 + wave] = b; }
        __syncthreads();
        s += wave / waves * waves;
        a = b = 0.f;
        for (uint32_t w = 0; w < waves; ++w) { a += s[w]; b += s[16 + w]; }
    }
    __device__ __forceinline__ void operator()(float& a) {
        a = wave_sum(a);
        if (waves == 1) return;
        float* s = scratch + 32u * (turn & 1u);
        ++turn;
        if (lane == 0) s[wave] = a;
        __syncthreads();
        s += wave / waves * waves;
        a = 0.f;
        for (uint32_t w = 0; w < waves; ++w) a += s[w];
    }
};

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// ---- route --------------------------------------------------------------------------------------------------
// A stable counting sort.  A wave takes strips of 64 consecutive slots; lanes with the same expert find each other by
// one ballot per bit of the expert number, so a slot's place among its equals in the strip is a population count, and
// the wave's running count of each expert sits in LDS.  Nothing depends on the order in which waves arrive.
// Few slots: one workgroup does it all in one launch.  More: one launch counts the slots of each expert in every block
// of kRouteBlock slots and one places them, every block adding up the counts of the blocks before it.  Many blocks:
// that sum, which grows with the square of the blocks, becomes a launch of its own.
// Bound by latency, not by bytes: 128 slots 2.7 us (a launch), 8192 over 256 experts 11.5 (two launches would take 9.3 on the
// GPU and 2 more on the host), 131072 12.6 (with the sum in a launch of its own 12.9, and 8 more on the host), 1048576 over
// 256 19.8 (adding up in every block: 32), of which 17 MB at the card's copy rate are 3.  Blocks of 2048 slots were faster up
// to 131072 (9 us) and slower above (27 at 524288), blocks of 8192 slower everywhere below a million.
constexpr uint32_t kRouteThreads = 1024, kRouteWaves = kRouteThreads / kWave;
constexpr uint32_t kRouteOneStrips = 8, kRouteStrips = 4;
constexpr uint32_t kRouteOne = kRouteThreads * kRouteOneStrips, kRouteBlock = kRouteThreads * kRouteStrips;
constexpr uint64_t kRouteSumMost = 16384;   // counts that a block adds up itself, at most
constexpr uint32_t kDropped = 0xffffffffu;
enum { kRouteAlone, kRouteSum, kRouteScanned };   // where a block's first rows come from

template <typename I>
__device__ __forceinline__ uint32_t slot_expert(const I* experts, uint32_t n, uint32_t slot, uint32_t num_experts) {
    if (slot >= n) return kDropped;
    const I id = experts[slot];
    return id >= 0 && id < (I)num_experts ? (uint32_t)id : kDropped;
}

// counts[expert * expert_step + block * block_step]
template <typename I>
__global__ __launch_bounds__(kRouteThreads) void route_count_kernel(const I* __restrict__ experts, uint32_t n, uint32_t num_experts,
                                                                    uint32_t* __restrict__ counts, uint32_t expert_step, uint32_t block_step) {
    __shared__ uint32_t hist[SAR_MAX_EXPERTS];
    const uint32_t tid = threadIdx.x, block = blockIdx.x;
    uint32_t key[kRouteStrips];
#pragma unroll
    for (uint32_t s = 0; s < kRouteStrips; ++s) key[s] = slot_expert(experts, n, block * kRouteBlock + s * kRouteThreads + tid, num_experts);
    if (tid < num_experts) hist[tid] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t s = 0; s < kRouteStrips; ++s)
        if (key[s] != kDropped) atomicAdd(&hist[key[s]], 1u);
    __syncthreads();
    if (tid < num_experts) counts[(uint64_t)tid * expert_step + (uint64_t)block * block_step] = hist[tid];
}

// One wave per expert: counts[expert][block] becomes the number of its slots in earlier blocks, totals[expert] all.
__global__ __launch_bounds__(kWave) void route_scan_kernel(uint32_t* __restrict__ counts, uint32_t* __restrict__ totals, uint32_t blocks) {
    uint32_t* const mine = counts + (uint64_t)blockIdx.x * blocks;
    const uint32_t lane = threadIdx.x;
    uint32_t before = 0;
    for (uint32_t b = 0; b < blocks; b += kWave) {
        const uint32_t v = b + lane < blocks ? mine[b + lane] : 0u;
        uint32_t sum = v;
        for (uint32_t d = 1; d < kWave; d <<= 1) {
            const uint32_t left = __shfl_up(sum, d, kWave);
            if (lane >= d) sum += left;
        }
        if (b + lane < blocks) mine[b + lane] = before + sum - v;
        before += __shfl(sum, kWave - 1, kWave);
    }
    if (lane == 0) totals[blockIdx.x] = before;
}

// Threads of one part of the sum over blocks: the experts, rounded up to whole waves and a divisor of the workgroup.
__host__ __device__ inline uint32_t route_part(uint32_t num_experts) {
    uint32_t part = kWave;
    while (part < num_experts) part *= 2;
    return part;
}

template <typename I, uint32_t STRIPS, int HOW>
__global__ __launch_bounds__(kRouteThreads) void route_place_kernel(const I* __restrict__ experts, uint32_t n, uint32_t num_experts,
                                                                    uint32_t key_bits, const uint32_t* __restrict__ counts,
                                                                    const uint32_t* __restrict__ totals, uint32_t blocks,
                                                                    int32_t* __restrict__ row_of_slot, int32_t* __restrict__ slot_of_row,
                                                                    int32_t* __restrict__ offsets) {
    __shared__ uint16_t seen[kRouteWaves * SAR_MAX_EXPERTS];   // slots of an expert: this wave's so far, then earlier waves'
    __shared__ uint32_t first[SAR_MAX_EXPERTS];
    __shared__ uint32_t part_before[HOW == kRouteSum ? kRouteThreads : 1], part_all[HOW == kRouteSum ? kRouteThreads : 1];
    __shared__ uint32_t wave_total[kRouteWaves];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wave = uniform(tid / kWave);
    const uint32_t begin = blockIdx.x * (kRouteThreads * STRIPS);
    uint16_t* const mine = seen + wave * num_experts;

    uint32_t key[STRIPS], place[STRIPS];
#pragma unroll
    for (uint32_t s = 0; s < STRIPS; ++s)
        key[s] = slot_expert(experts, n, begin + (wave * STRIPS + s) * kWave + lane, num_experts);
    uint32_t sum = 0, before = 0;                                // slots of expert `tid`: all, and in earlier blocks
    if (HOW == kRouteScanned && tid < num_experts) {
        sum = totals[tid];
        before = counts[(uint64_t)tid * blocks + blockIdx.x];
    }
    const uint32_t part = HOW == kRouteSum ? route_part(num_experts) : 1u;
    if (HOW == kRouteSum) {
        const uint32_t expert = tid & (part - 1u), parts = kRouteThreads / part;
        uint32_t early = 0, all = 0;
        if (expert < num_experts) {
#pragma unroll 8
            for (uint32_t b = tid / part; b < blocks; b += parts) {
                const uint32_t v = counts[(uint64_t)b * num_experts + expert];
                all += v;
                early += b < blockIdx.x ? v : 0u;
            }
        }
        part_before[tid] = early;
        part_all[tid] = all;
    }
    for (uint32_t i = lane; i < num_experts; i += kWave) mine[i] = 0;
    const uint64_t below = (1ull << lane) - 1ull;
#pragma unroll
    for (uint32_t s = 0; s < STRIPS; ++s) {
        const bool in = key[s] != kDropped;
        uint64_t equal = __ballot(in);
        for (uint32_t b = 0; b < key_bits; ++b) {
            const uint64_t set = __ballot((key[s] >> b) & 1u);
            equal &= (key[s] >> b) & 1u ? set : ~set;
        }
        const uint32_t rank = (uint32_t)__popcll(equal & below);
        // one wave's LDS accesses are done in order: every lane has read before the first of its equals writes
        const uint32_t earlier = in ? mine[key[s]] : 0u;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (in && rank == 0) mine[key[s]] = (uint16_t)(earlier + (uint32_t)__popcll(equal));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        place[s] = earlier + rank;
    }
    __syncthreads();

    if (tid < num_experts) {
        uint32_t v[kRouteWaves], so_far = 0;
#pragma unroll
        for (uint32_t w = 0; w < kRouteWaves; ++w) v[w] = seen[w * num_experts + tid];
#pragma unroll
        for (uint32_t w = 0; w < kRouteWaves; ++w) {
            seen[w * num_experts + tid] = (uint16_t)so_far;
            so_far += v[w];
        }
        if (HOW == kRouteAlone) sum = so_far;
        if (HOW == kRouteSum)
            for (uint32_t p = tid; p < kRouteThreads; p += part) { sum += part_all[p]; before += part_before[p]; }
    }
    uint32_t upto = sum;                                         // inclusive sum over the experts, wave by wave
    for (uint32_t d = 1; d < kWave; d <<= 1) {
        const uint32_t left = __shfl_up(upto, d, kWave);
        if (lane >= d) upto += left;
    }
    if (lane == kWave - 1) wave_total[wave] = upto;
    __syncthreads();
    uint32_t total = 0;
    for (uint32_t w = 0; w < kRouteWaves; ++w) {
        if (w < wave) upto += wave_total[w];
        total += wave_total[w];
    }
    if (tid < num_experts) {
        first[tid] = upto - sum + before;
        if (blockIdx.x == 0) offsets[tid] = (int32_t)(upto - sum);
    }
    if (blockIdx.x == 0 && tid == 0) offsets[num_experts] = (int32_t)total;
    __syncthreads();

#pragma unroll
    for (uint32_t s = 0; s < STRIPS; ++s) {
        const uint32_t slot = begin + (wave * STRIPS + s) * kWave + lane;
        if (slot >= n) continue;
        const bool in = key[s] != kDropped;
        const uint32_t row = in ? first[key[s]] + seen[wave * num_experts + key[s]] + place[s] : kDropped;
        row_of_slot[slot] = (int32_t)row;
        if (row < n) slot_of_row[row] = (int32_t)slot;            // (expert numbers that change between the launches)
        if (slot >= total) slot_of_row[slot] = -1;               // the rows behind the last one
    }
}

// ---- dispatch, combine --------------------------------------------------------------------------------------
// A wave takes one token (and 64 vectors of its row).  Lane k holds the row and the weight of choice k;
// the choices that were not dropped are the bits of a ballot, walked in order with the row number in a scalar register.
// Row numbers come from memory and are held against the number of rows before they become an address.
// Bound by HBM: 16384 tokens of 2048 in bf16, eight choices (0.6 GB): dispatch 105 us, 5.7 TB/s (a torch copy of that size
// 5.1), combine 101 us, 6.0 TB/s.  Consecutive tokens per XCD instead of round robin changed nothing (231 against 236 us for
// both).
constexpr uint32_t kMoveThreads = 256, kMoveWaves = kMoveThreads / kWave;

struct MoveArgs {
    const char* in;          // dispatch: tokens; combine: rows; backward: grad
    const char* rows;        // backward: rows
    char* out;               // dispatch: rows; combine: tokens; backward: grad_rows (may be null)
    const char* weights;     // null: all one
    char* grad_weights;
    const int32_t* row_of_slot;
    const int32_t* total;    // number of rows in use
    uint64_t tokens;
    uint32_t topk, nrows, dim, nvec, row_bytes, weights_f32;
};

// Zeros in the rows nobody was sent to: row total + token, and every `tokens`-th behind it.
template <int DT, int VE, int U, bool NT>
__device__ __forceinline__ void zero_rows(const MoveArgs& a, uint64_t token, uint32_t v0) {
    uint32_t total = uniform((uint32_t)*a.total);
    if (total > a.nrows) total = a.nrows;
    for (uint64_t row = total + token; row < a.nrows; row += a.tokens) {
        char* const to = a.out + row * a.row_bytes;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Place<DT, VE> p(v0 + u * kWave, a.nvec, a.dim);
            if (p.in) store<DT, VE, NT>(to, p.byte(), typename Raw<DT, VE>::T{});
        }
    }
}

__device__ __forceinline__ uint32_t lane_value(uint32_t x, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, lane); }
__device__ __forceinline__ float lane_value(float x, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane)); }

template <int DT, int VE, bool NT, bool WEIGHTED>
__global__ __launch_bounds__(kMoveThreads) void dispatch_kernel(const MoveArgs a) {
    typedef typename Raw<DT, VE>::T R;
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x / kWave), vec = blockIdx.x * kWave + lane;
    const Place<DT, VE> p(vec, a.nvec, a.dim);
    for (uint64_t token = (uint64_t)blockIdx.y * kMoveWaves + wave; token < a.tokens; token += (uint64_t)gridDim.y * kMoveWaves) {
        const uint64_t slot = token * a.topk + min(lane, a.topk - 1);
        const uint32_t listed = (uint32_t)a.row_of_slot[slot];
        float weight = 1.f;
        if (WEIGHTED) weight = load_one<DT>(a.weights, a.weights_f32, slot);
        const R v = load<DT, VE>(a.in + token * a.row_bytes, p.byte());
        for (uint64_t left = __ballot(lane < a.topk && listed < a.nrows); left; left &= left - 1) {
            const int k = __builtin_ctzll(left);
            char* const to = a.out + (uint64_t)lane_value(listed, k) * a.row_bytes;
            R r = v;
            if constexpr (WEIGHTED) {
                const float w = lane_value(weight, k);
                float x[VE];
                unpack<DT, VE>(r, x);
#pragma unroll
                for (int i = 0; i < VE; ++i) x[i] *= w;
                r = pack<DT, VE>(x);
            }
            if (p.in) store<DT, VE, NT>(to, p.byte(), r);
        }
        zero_rows<DT, VE, 1, NT>(a, token, vec);
    }
}

// The sum is kept in 32 bits and taken in the order of the choices.
template <int DT, int VE, bool NT>
__global__ __launch_bounds__(kMoveThreads) void combine_kernel(const MoveArgs a) {
    struct Row { typename Raw<DT, VE>::T v; float w; };
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x / kWave);
    const Place<DT, VE> p(blockIdx.x * kWave + lane, a.nvec, a.dim);
    for (uint64_t token = (uint64_t)blockIdx.y * kMoveWaves + wave; token < a.tokens; token += (uint64_t)gridDim.y * kMoveWaves) {
        const uint64_t slot = token * a.topk + min(lane, a.topk - 1);
        const uint32_t listed = (uint32_t)a.row_of_slot[slot];
        float weight = 1.f;
        if (a.weights) weight = load_one<DT>(a.weights, a.weights_f32, slot);
        float sum[VE] = {};
        uint64_t left = __ballot(lane < a.topk && listed < a.nrows);
        in_batches<8>((uint32_t)__popcll(left),
                      [&](uint32_t) {
                          const int k = __builtin_ctzll(left);
                          left &= left - 1;
                          return Row{load<DT, VE, NT>(a.in + (uint64_t)lane_value(listed, k) * a.row_bytes, p.byte()), lane_value(weight, k)};
                      },
                      [&](const Row& r) {
                          float x[VE];
                          unpack<DT, VE>(r.v, x);
#pragma unroll
                          for (int i = 0; i < VE; ++i) sum[i] = fmaf(r.w, x[i], sum[i]);
                      });
        if (p.in) store<DT, VE, NT>(a.out + token * a.row_bytes, p.byte(), pack<DT, VE>(sum));
    }
}

// Both gradients in one pass over the rows: a token's gradient row stays in registers while its rows go by, each read
// once for its dot product (summed in 32 bits, kept in the lane of its choice) and written once.  SHARE waves take one
// token's segments in turn where the rows are long; their dot products are added in wave order.  Bound by HBM: 16384
// tokens of 4096 in bf16, four choices (1.2 GB) 222 us, 5.4 TB/s.
template <int DT, int VE, int U, int SHARE, bool NT>
__global__ __launch_bounds__(kMoveThreads) void combine_backward_kernel(const MoveArgs a) {
    typedef typename Raw<DT, VE>::T R;
    __shared__ float dots[kMoveWaves][kWave];
    const uint32_t lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x / kWave);
    const uint32_t part = wave % SHARE;
    constexpr uint32_t kTokens = kMoveWaves / SHARE;            // tokens a workgroup has in hand
    struct Row { R v[U]; float w; int k; uint64_t at; };
    for (uint64_t base = (uint64_t)blockIdx.x * kTokens; base < a.tokens; base += (uint64_t)gridDim.x * kTokens) {
        const uint64_t token = base + wave / SHARE;
        if (SHARE > 1 || token < a.tokens) {
            const uint64_t slot = token * a.topk + min(lane, a.topk - 1);
            const uint32_t listed = (uint32_t)a.row_of_slot[slot];
            const float weight = load_one<DT>(a.weights, a.weights_f32, slot);
            const uint64_t present = __ballot(lane < a.topk && listed < a.nrows);
            const uint32_t count = (uint32_t)__popcll(present);
            const char* const grad = a.in + token * a.row_bytes;
            float dot = 0.f;                                     // of choice `lane`
            for (uint32_t seg = part * (U * kWave); seg < a.nvec; seg += SHARE * U * kWave) {
                const uint32_t v0 = seg + lane;
                float g[U][VE];
#pragma unroll
                for (int u = 0; u < U; ++u) unpack<DT, VE>(load<DT, VE, NT>(grad, Place<DT, VE>(v0 + u * kWave, a.nvec, a.dim).byte()), g[u]);
                uint64_t left = present;
                auto ld = [&](uint32_t) {
                    Row r;
                    r.k = __builtin_ctzll(left);
                    left &= left - 1;
                    r.at = (uint64_t)lane_value(listed, r.k) * a.row_bytes;
                    r.w = lane_value(weight, r.k);
#pragma unroll
                    for (int u = 0; u < U; ++u) r.v[u] = load<DT, VE, NT>(a.rows + r.at, Place<DT, VE>(v0 + u * kWave, a.nvec, a.dim).byte());
                    return r;
                };
                auto use = [&](const Row& r) {
                    float s = 0.f;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const Place<DT, VE> p(v0 + u * kWave, a.nvec, a.dim);
                        float y[VE], x[VE];
                        unpack<DT, VE>(r.v[u], y);
#pragma unroll
                        for (int i = 0; i < VE; ++i) {
                            s = (uint32_t)i >= p.skip ? fmaf(g[u][i], y[i], s) : s;
                            x[i] = g[u][i] * r.w;
                        }
                        if (a.out && p.in) store<DT, VE, NT>(a.out + r.at, p.byte(), pack<DT, VE>(x));
                    }
                    s = wave_sum(s);
                    if ((int)lane == r.k) dot += s;
                };
                in_batches<2>(count, ld, use);
                if (a.out) zero_rows<DT, VE, U, NT>(a, token, v0);
            }
            if (SHARE > 1) dots[wave][lane] = dot;
            else if (lane < a.topk) store_one<DT>(a.grad_weights, a.weights_f32, slot, dot);
        }
        if (SHARE > 1) {
            __syncthreads();
            if (part == 0 && lane < a.topk) {
                float dot = 0.f;
                for (uint32_t p = 0; p < SHARE; ++p) dot += dots[wave + p][lane];
                store_one<DT>(a.grad_weights, a.weights_f32, token * a.topk + lane, dot);
            }
            __syncthreads();
        }
    }
}

// ---- sum over the ranks, norms, gate, residual ----------------------------------------------------------------
// A workgroup takes one token; its row stays in registers in 32 bits from the sum over the ranks to the last norm, one
// 16-byte vector a thread as long as 1024 threads reach.  Two vectors, from eight ranks in bf16: 6.4 us against 5.1 for 16
// tokens of 4096, 15.8 against 14.3 for 1024 of 2048, level to 5 % slower from 302 MB on, but 16 to 18 % faster in the three
// calls measured that move 151 MB (1024 of 4096: 27.2 against 32.6); that is not explained, and no rule is made of it.  Bound
// by HBM: 8192 tokens of 4096 in bf16 with a copy of the result for every rank (1.2 GB) 205 us, 5.9 TB/s.  A grid that stays
// and keeps its weights in registers took 240 where this took 228.
struct NormArgs {
    const char* partials[SAR_MAX_RANKS];
    const char* residual;
    const char* pre;
    const char* post;
    const char* gate;
    char* hidden;
    char* normed;
    float* total;
    float* stats;
    uint64_t tokens, copy_bytes;
    uint32_t dim, nvec, row_bytes, sources, copies, gate_kind, pre_f32, post_f32, gate_f32;
    float eps, residual_scale, inv_dim;
};

constexpr uint32_t kNormThreads = 1024;
constexpr uint32_t kRowsThreads = 512;   // backward pass: workgroups of short rows take several of them up to here

// A thread's place in its row: it takes vectors at, at + step, ...
struct RowPart { uint32_t at, step; };

template <int DT, int VE, int V> struct Vectors { typename Raw<DT, VE>::T v[V]; };

template <int DT, int VE, int V, bool NT = false>
__device__ __forceinline__ Vectors<DT, VE, V> load_row(const char* row, const NormArgs& a, RowPart r) {
    Vectors<DT, VE, V> x;
#pragma unroll
    for (int v = 0; v < V; ++v) x.v[v] = load<DT, VE, NT>(row, Place<DT, VE>(r.at + v * r.step, a.nvec, a.dim).byte());
    return x;
}
template <int DT, int VE, int V>
__device__ __forceinline__ void load_params(const char* p, bool f32, const NormArgs& a, RowPart r, float (&x)[V][VE]) {
#pragma unroll
    for (int v = 0; v < V; ++v) load_param<DT, VE>(p, f32, Place<DT, VE>(r.at + v * r.step, a.nvec, a.dim).elem, x[v]);
}
template <int V, int VE>
__device__ __forceinline__ void set(float (&x)[V][VE], float value) {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < VE; ++i) x[v][i] = value;
}
template <int V, int VE>
__device__ __forceinline__ void copy(float (&x)[V][VE], const float (&y)[V][VE]) {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < VE; ++i) x[v][i] = y[v][i];
}
template <int DT, int VE, int V>
__device__ __forceinline__ void add_row(float (&x)[V][VE], const Vectors<DT, VE, V>& r) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float y[VE];
        unpack<DT, VE>(r.v[v], y);
#pragma unroll
        for (int i = 0; i < VE; ++i) x[v][i] += y[i];
    }
}
// `count` copies of a row, `step` bytes apart
template <int DT, int VE, int V, bool NT>
__device__ __forceinline__ void store_row(char* to, uint64_t step, uint32_t count, const float (&x)[V][VE], const NormArgs& a, RowPart r) {
    Vectors<DT, VE, V> out;
#pragma unroll
    for (int v = 0; v < V; ++v) out.v[v] = pack<DT, VE>(x[v]);
    for (uint32_t c = 0; c < count; ++c, to += step) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Place<DT, VE> p(r.at + v * r.step, a.nvec, a.dim);
            if (p.in) store<DT, VE, NT>(to, p.byte(), out.v[v]);
        }
    }
}
// a row in 32 bits, or in DT if f32 is false
template <int DT, int VE, int V>
__device__ __forceinline__ void store_params(char* to, bool f32, const float (&x)[V][VE], const NormArgs& a, RowPart r) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const Place<DT, VE> p(r.at + v * r.step, a.nvec, a.dim);
        if (!p.in) continue;
        if (DT == SAR_F32 || f32) {
            if constexpr (VE == 1) store<SAR_F32, 1>(to, p.elem * 4u, __float_as_uint(x[v][0]));
            else {
#pragma unroll
                for (int q = 0; q < VE / 4; ++q) store<SAR_F32, 4>(to, p.elem * 4u + 16u * q, pack<SAR_F32, 4>(x[v] + 4 * q));
            }
        } else {
            store<DT, VE>(to, p.byte(), pack<DT, VE>(x[v]));
        }
    }
}
// this thread's part of the sum over a row of x * y, doubled elements once
template <int DT, int VE, int V>
__device__ __forceinline__ float dot_row(const float (&x)[V][VE], const float (&y)[V][VE], const NormArgs& a, RowPart r) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const Place<DT, VE> p(r.at + v * r.step, a.nvec, a.dim);
#pragma unroll
        for (int i = 0; i < VE; ++i) s = (uint32_t)i >= p.skip ? fmaf(x[v][i], y[v][i], s) : s;
    }
    return s;
}

template <int DT, int VE, int V, bool ONE, bool NT>
__global__ __launch_bounds__(kNormThreads) void reduce_norm_kernel(const NormArgs a) {
    constexpr uint32_t ES = ElemSize<DT>::value;
    constexpr bool kEarly = V * VE <= 8;    // weights for the first half are loaded beside the row where there are registers
    __shared__ float scratch[64];
    const RowPart r{threadIdx.x, blockDim.x};
    RowSum sum{scratch, 0u, blockDim.x / kWave, uniform(threadIdx.x / kWave), threadIdx.x & (kWave - 1)};
    float post[V][VE], pre[V][VE], gate[V][VE];
    for (uint64_t token = blockIdx.x; token < a.tokens; token += gridDim.x) {
        const uint64_t at = token * a.row_bytes;
        const auto res = load_row<DT, VE, V>(a.residual + at, a, r);
        if (kEarly) {
            if (a.post) load_params<DT, VE, V>(a.post, a.post_f32, a, r, post);
            if (a.gate_kind == SAR_GATE_CHANNEL) load_params<DT, VE, V>(a.gate, a.gate_f32, a, r, gate);
        }
        if (a.gate_kind == SAR_GATE_FULL) load_params<DT, VE, V>(a.gate + token * a.dim * (a.gate_f32 ? 4u : ES), a.gate_f32, a, r, gate);
        if (a.gate_kind == SAR_GATE_TOKEN) set(gate, load_one<DT>(a.gate, a.gate_f32, token));
        float x[V][VE];
        set(x, 0.f);
        in_batches<ONE ? 1 : 8 / V>(ONE ? 1u : a.sources, [&](uint32_t s) { return load_row<DT, VE, V, NT>(a.partials[s] + at, a, r); },
                                    [&](const Vectors<DT, VE, V>& p) { add_row<DT, VE, V>(x, p); });
        if (a.total) store_params<DT, VE, V>((char*)(a.total + token * a.dim), true, x, a, r);
        float r1 = 1.f;
        if (a.post) {
            r1 = dot_row<DT, VE, V>(x, x, a, r);
            sum(r1);
            r1 = rsqrtf(fmaf(r1, a.inv_dim, a.eps));
            if (!kEarly) load_params<DT, VE, V>(a.post, a.post_f32, a, r, post);
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < VE; ++i) x[v][i] = x[v][i] * r1 * post[v][i];
        }
        if (!kEarly && a.gate_kind == SAR_GATE_CHANNEL) load_params<DT, VE, V>(a.gate, a.gate_f32, a, r, gate);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float h[VE];
            unpack<DT, VE>(res.v[v], h);
#pragma unroll
            for (int i = 0; i < VE; ++i) x[v][i] = fmaf(a.residual_scale, h[i], a.gate_kind == SAR_GATE_NONE ? x[v][i] : gate[v][i] * x[v][i]);
        }
        if (a.hidden) store_row<DT, VE, V, false>(a.hidden + at, 0, 1, x, a, r);
        float r2 = 1.f;
        if (a.pre) {
            r2 = dot_row<DT, VE, V>(x, x, a, r);
            sum(r2);
            r2 = rsqrtf(fmaf(r2, a.inv_dim, a.eps));
            load_params<DT, VE, V>(a.pre, a.pre_f32, a, r, pre);
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < VE; ++i) x[v][i] = x[v][i] * r2 * pre[v][i];
            store_row<DT, VE, V, NT>(a.normed + at, a.copy_bytes, a.copies, x, a, r);
        }
        if (a.stats && threadIdx.x == 0) { a.stats[token] = r1; a.stats[a.tokens + token] = r2; }
    }
}

// With yhat = y r1, u = yhat post, hidden = s residual + g u, hhat = hidden r2, G = sum of the copies' gradients:
//   d hidden   = grad_hidden + r2 (G pre - hhat mean(G pre hhat))      d residual = s d hidden       d pre  = sum_t G hhat
//   d u        = g d hidden                                            d g = d hidden u, summed      d post = sum_t du yhat
//   d partials = r1 (du post - yhat mean(du post yhat))
// hidden is computed again from y and the residual, so nothing that was rounded comes back.  A workgroup walks over
// tokens and keeps the column sums in registers; they leave as one row of sums per workgroup, added up by
// column_sum_kernel in a fixed order; a single workgroup writes the gradients itself.
// Bound by HBM where ranks are many: 4096 tokens of 4096 in bf16 to and from eight ranks (0.73 GB) 133 us, 5.5 TB/s; by the
// two sums over a row that every token waits for where they are not: one row in, one out 53 us for 0.23 GB.  Loading the next
// token ahead cost registers that were spilled (79 us), as did five or six waves a SIMD (71, 93).
struct NormBackwardArgs {
    NormArgs f;
    const char* total;
    const char* grad_hidden;
    const char* grad_normed;
    char* grad_partials;
    char* grad_residual;
    char* grad_gate;                   // per token or full (a channel gate's gradient is a column sum)
    float* columns;                    // [workgroup][3][dim], unless there is only one
    char* grad_weights[3];             // of pre, post and a channel gate: null = not wanted
    uint32_t weights_f32[3], total_f32;
    uint32_t row_threads;              // threads of one row
};

// A thread's column sums, in registers or, for rows that leave none, in LDS (a thread touches its own only).
template <int V, int VE, bool LDS> struct Columns {
    float x[V][VE];
    __device__ __forceinline__ void init(f4*) { set(x, 0.f); }
    __device__ __forceinline__ void add(int v, const float (&a)[VE], const float (&b)[VE]) {
#pragma unroll
        for (int i = 0; i < VE; ++i) x[v][i] = fmaf(a[i], b[i], x[v][i]);
    }
    __device__ __forceinline__ void get(float (&y)[V][VE]) const {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < VE; ++i) y[v][i] = x[v][i];
    }
};
template <int V, int VE> struct Columns<V, VE, true> {
    f4* mine;          // entry of this thread; the next vector of four is kNormThreads further on
    __device__ __forceinline__ void init(f4* lds) {
        mine = lds + threadIdx.x;
#pragma unroll
        for (int q = 0; q < V * VE / 4; ++q) mine[q * kNormThreads] = f4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void add(int v, const float (&a)[VE], const float (&b)[VE]) {
#pragma unroll
        for (int q = 0; q < VE / 4; ++q) {
            f4 m = mine[(v * (VE / 4) + q) * kNormThreads];
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = fmaf(a[4 * q + i], b[4 * q + i], m[i]);
            mine[(v * (VE / 4) + q) * kNormThreads] = m;
        }
    }
    __device__ __forceinline__ void get(float (&y)[V][VE]) const {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int q = 0; q < VE / 4; ++q) {
                const f4 m = mine[(v * (VE / 4) + q) * kNormThreads];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[v][4 * q + i] = m[i];
            }
    }
};

template <int DT, int VE, int V, bool ONE, bool NT>
__global__ __launch_bounds__(kNormThreads) void reduce_norm_backward_kernel(const NormBackwardArgs b) {
    constexpr uint32_t ES = ElemSize<DT>::value;
    constexpr uint32_t kMost = V == 1 ? kRowsThreads : 0u;              // threads of a workgroup that takes several tokens
    __shared__ float scratch[64];
    __shared__ float rows[kMost ? kMost * VE : 1];
    const NormArgs& a = b.f;
    const uint32_t many = blockDim.x / b.row_threads, mine = many == 1 ? 0u : uniform(threadIdx.x / b.row_threads);
    const RowPart r{threadIdx.x - mine * b.row_threads, b.row_threads};
    RowSum sum{scratch, 0u, b.row_threads / kWave, uniform(threadIdx.x / kWave), threadIdx.x & (kWave - 1)};
    // 16 elements a thread: two of the three column sums (128 KB) stay in LDS (206 -> 131 us for 1000 tokens of 16384).  The
    // compiler spills even so, 76 registers in bf16, 49 in f16 and 64 in f32 (228, 200 and 260 bytes a lane): from and to
    // four ranks those 1000 tokens in bf16 take 161 us for 476 MB of their own and some 300 MB of scratch.  Eight elements: 5 in
    // bf16 and 2 in f16, f32 none.
    constexpr bool kInLds = V * VE > 8;
    __shared__ f4 lds[kInLds ? 2 * (V * VE / 4) * kNormThreads : 1];
    Columns<V, VE, kInLds> col_pre, col_post;
    Columns<V, VE, false> col_gate;
    col_pre.init(lds), col_post.init(lds + (kInLds ? V * VE / 4 * kNormThreads : 0)), col_gate.init(nullptr);
    // One row in, one row out: nothing to batch, so the weights stay in registers from token to token (4096 tokens of 4096
    // 62 -> 50 us).  With eight rows to write it was slower so (20000 of 2048: 219 us against 240).
    constexpr bool kKeep = ONE;
    constexpr int kKept = kKeep ? V : 1, kKeptVE = kKeep ? VE : 1;
    float kept_pre[kKept][kKeptVE], kept_post[kKept][kKeptVE], kept_gate[kKept][kKeptVE];
    if constexpr (kKeep) {
        if (a.pre) load_params<DT, VE, V>(a.pre, a.pre_f32, a, r, kept_pre);
        if (a.post) load_params<DT, VE, V>(a.post, a.post_f32, a, r, kept_post);
        else set(kept_post, 1.f);
        if (a.gate_kind == SAR_GATE_CHANNEL) load_params<DT, VE, V>(a.gate, a.gate_f32, a, r, kept_gate);
    }
    for (uint64_t first = (uint64_t)blockIdx.x * many; first < a.tokens; first += (uint64_t)gridDim.x * many) {
        const bool in = first + mine < a.tokens;                        // the sums are the whole workgroup's affair
        const uint64_t token = in ? first + mine : a.tokens - 1;
        const uint64_t at = token * a.row_bytes;
        const float r1 = a.stats[token], r2 = a.stats[a.tokens + token];
        const float token_gate = a.gate_kind == SAR_GATE_TOKEN ? load_one<DT>(a.gate, a.gate_f32, token) : 1.f;
        const auto res = load_row<DT, VE, V, NT>(a.residual + at, a, r);
        Vectors<DT, VE, V> gh{};
        if (b.grad_hidden) gh = load_row<DT, VE, V, NT>(b.grad_hidden + at, a, r);
        float y[V][VE];      // yhat (y without a norm there)
        load_params<DT, VE, V>(b.total + token * a.dim * (b.total_f32 ? 4u : ES), b.total_f32, a, r, y);
        float d[V][VE];      // G, then G pre, then d hidden
        set(d, 0.f);
        if (b.grad_normed)
            in_batches<ONE ? 1 : kInLds ? 8 / V / 2 : V == 1 ? 4 : 8 / V>(ONE ? 1u : a.copies, [&](uint32_t c) { return load_row<DT, VE, V, NT>(b.grad_normed + at + c * a.copy_bytes, a, r); },
                       [&](const Vectors<DT, VE, V>& p) { add_row<DT, VE, V>(d, p); });
        float post[V][VE], gate[V][VE], h[V][VE];      // h: hhat
        auto load_gates = [&]() {
            if constexpr (kKeep) copy(post, kept_post);
            else if (a.post) load_params<DT, VE, V>(a.post, a.post_f32, a, r, post);
            else set(post, 1.f);
            if (a.gate_kind == SAR_GATE_CHANNEL) {
                if constexpr (kKeep) copy(gate, kept_gate);
                else load_params<DT, VE, V>(a.gate, a.gate_f32, a, r, gate);
            } else if (a.gate_kind == SAR_GATE_FULL) {
                load_params<DT, VE, V>(a.gate + token * a.dim * (a.gate_f32 ? 4u : ES), a.gate_f32, a, r, gate);
            } else {
                set(gate, token_gate);
            }
        };
        load_gates();
#pragma unroll
        for (int v = 0; v < V; ++v) {
            unpack<DT, VE>(res.v[v], h[v]);
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                y[v][i] *= r1;
                h[v][i] = fmaf(a.residual_scale, h[v][i], gate[v][i] * (y[v][i] * post[v][i])) * r2;
            }
        }
        if (b.grad_normed) {
            float pre[V][VE];
            if constexpr (kKeep) copy(pre, kept_pre);
            else load_params<DT, VE, V>(a.pre, a.pre_f32, a, r, pre);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (in) col_pre.add(v, d[v], h[v]);
#pragma unroll
                for (int i = 0; i < VE; ++i) d[v][i] *= pre[v][i];
            }
            float mean = dot_row<DT, VE, V>(d, h, a, r);
            sum(mean);
            mean *= a.inv_dim;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < VE; ++i) d[v][i] = r2 * fmaf(-h[v][i], mean, d[v][i]);
        }
        if (b.grad_hidden) add_row<DT, VE, V>(d, gh);
        if (b.grad_residual && in) {
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < VE; ++i) h[v][i] = a.residual_scale * d[v][i];
            store_row<DT, VE, V, NT>(b.grad_residual + at, 0, 1, h, a, r);
        }
        float gate_dot = 0.f;
        if (kInLds) load_gates();                      // again, from the cache: kept they would be spilled too
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Place<DT, VE> p(r.at + v * r.step, a.nvec, a.dim);
#pragma unroll
            for (int i = 0; i < VE; ++i) h[v][i] = y[v][i] * post[v][i];       // u
            if (in) col_gate.add(v, d[v], h[v]);
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                h[v][i] *= d[v][i];                                          // gradient of the gate
                gate_dot += (uint32_t)i >= p.skip ? h[v][i] : 0.f;
                d[v][i] *= gate[v][i];
            }
            if (in) col_post.add(v, d[v], y[v]);
#pragma unroll
            for (int i = 0; i < VE; ++i) d[v][i] *= post[v][i];
        }
        if (a.gate_kind == SAR_GATE_FULL && b.grad_gate && in) store_params<DT, VE, V>(b.grad_gate + token * a.dim * (a.gate_f32 ? 4u : ES), a.gate_f32, h, a, r);
        if (a.post) {
            float mean = dot_row<DT, VE, V>(d, y, a, r);
            sum(mean, gate_dot);
            mean *= a.inv_dim;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < VE; ++i) d[v][i] = r1 * fmaf(-y[v][i], mean, d[v][i]);
        } else if (a.gate_kind == SAR_GATE_TOKEN) {
            sum(gate_dot);
        }
        if (a.gate_kind == SAR_GATE_TOKEN && b.grad_gate && in && r.at == 0) store_one<DT>(b.grad_gate, a.gate_f32, token, gate_dot);
        if (b.grad_partials && in) store_row<DT, VE, V, NT>(b.grad_partials + at, a.copy_bytes, a.sources, d, a, r);
    }
    auto leave = [&](const auto& columns, uint32_t which) {
        float x[V][VE];
        columns.get(x);
        if constexpr (kMost != 0u) {
            if (many > 1) {                                              // the rows' sums, in their order
                __syncthreads();
#pragma unroll
                for (int i = 0; i < VE; ++i) rows[threadIdx.x * VE + i] = x[0][i];
                __syncthreads();
                if (mine) return;
                for (uint32_t m = 1; m < many; ++m)
#pragma unroll
                    for (int i = 0; i < VE; ++i) x[0][i] += rows[(m * r.step + r.at) * VE + i];
            }
        }
        if (gridDim.x == 1) store_params<DT, VE, V>(b.grad_weights[which], b.weights_f32[which], x, a, r);
        else store_params<DT, VE, V>((char*)(b.columns + ((uint64_t)blockIdx.x * 3u + which) * a.dim), true, x, a, r);
    };
    if (b.grad_weights[0]) leave(col_pre, 0);
    if (b.grad_weights[1]) leave(col_post, 1);
    if (b.grad_weights[2]) leave(col_gate, 2);
}

// Adds the workgroups' rows of column sums: 32 columns a workgroup, 32 groups of threads taking every 32nd row, then in
// the groups' order.
struct ColumnArgs {
    const float* columns;
    char* out[3];
    uint32_t f32[3];
    uint32_t rows, dim;
};
template <int DT>
__global__ __launch_bounds__(1024) void column_sum_kernel(const ColumnArgs a) {
    __shared__ float part[32][33];
    const uint32_t which = blockIdx.y, lane = threadIdx.x & 31u, group = threadIdx.x / 32u;
    if (!a.out[which]) return;
    const uint32_t col = blockIdx.x * 32u + lane;
    float s = 0.f;
    if (col < a.dim) {
        const float* from = a.columns + which * a.dim + col;
#pragma unroll 8
        for (uint32_t r = group; r < a.rows; r += 32u) s += from[(uint64_t)r * 3u * a.dim];
    }
    part[group][lane] = s;
    __syncthreads();
    if (group == 0 && col < a.dim) {
        s = 0.f;
#pragma unroll
        for (int g = 0; g < 32; ++g) s += part[g][lane];
        store_one<DT>(a.out[which], a.f32[which], col, s);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------

// Makes `device` current for a call and puts the caller's device back.
class OnDevice {
public:
    explicit OnDevice(int device) {
        err_ = hipGetDevice(&before_);
        if (err_ == hipSuccess && before_ != device) { err_ = hipSetDevice(device); moved_ = err_ == hipSuccess; }
    }
    ~OnDevice() { if (moved_) (void)hipSetDevice(before_); }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    hipError_t error() const { return err_; }
private:
    int before_ = 0;
    bool moved_ = false;
    hipError_t err_;
};

int refuse(const char* why) { return set_error(SAR_EINVAL, why); }
int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? (int)SAR_OK : set_error(SAR_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}
int not_current(int device, hipError_t e) {
    (void)hipGetLastError();
    return set_error(e == hipErrorNoDevice || e == hipErrorInvalidDevice ? SAR_ENODEV : SAR_EHIP,
                     "device " + std::to_string(device) + ": " + hipGetErrorString(e));
}

bool known_dtype(int dt) { return dt == SAR_F32 || dt == SAR_F16 || dt == SAR_BF16; }
uint32_t elem_size(int dt) { return dt == SAR_F32 ? 4u : 2u; }
bool aligned(const void* p, uint64_t to) { return (uintptr_t)p % to == 0; }

// calls f(integral_constant<int, DT>) for the dtype
template <class F> void with_dtype(int dt, F&& f) {
    if (dt == SAR_F32) f(std::integral_constant<int, SAR_F32>{});
    else if (dt == SAR_F16) f(std::integral_constant<int, SAR_F16>{});
    else f(std::integral_constant<int, SAR_BF16>{});
}

uint64_t route_blocks(uint64_t n) { return (n + kRouteBlock - 1) / kRouteBlock; }

template <typename I>
void launch_route(hipStream_t st, const void* experts, uint32_t n, uint32_t num_experts, int32_t* row_of_slot, int32_t* slot_of_row,
                  int32_t* offsets, uint32_t* workspace) {
    const I* ids = (const I*)experts;
    uint32_t bits = 0;
    while ((1u << bits) < num_experts) ++bits;
    if (n <= kRouteOne) {
        auto alone = [&](auto strips) {
            route_place_kernel<I, decltype(strips)::value, kRouteAlone><<<1, kRouteThreads, 0, st>>>(ids, n, num_experts, bits, nullptr, nullptr, 1, row_of_slot, slot_of_row, offsets);
        };
        if (n <= kRouteThreads) alone(std::integral_constant<uint32_t, 1>{});
        else if (n <= 4 * kRouteThreads) alone(std::integral_constant<uint32_t, 4>{});
        else alone(std::integral_constant<uint32_t, kRouteOneStrips>{});
        return;
    }
    const uint32_t blocks = (uint32_t)route_blocks(n);
    if (blocks * (uint64_t)route_part(num_experts) <= kRouteSumMost) {
        uint32_t* const counts = workspace;
        route_count_kernel<I><<<blocks, kRouteThreads, 0, st>>>(ids, n, num_experts, counts, 1, num_experts);
        route_place_kernel<I, kRouteStrips, kRouteSum><<<blocks, kRouteThreads, 0, st>>>(ids, n, num_experts, bits, counts, nullptr, blocks, row_of_slot, slot_of_row, offsets);
        return;
    }
    uint32_t* const totals = workspace;
    uint32_t* const counts = workspace + num_experts;
    route_count_kernel<I><<<blocks, kRouteThreads, 0, st>>>(ids, n, num_experts, counts, blocks, 1);
    route_scan_kernel<<<num_experts, kWave, 0, st>>>(counts, totals, blocks);
    route_place_kernel<I, kRouteStrips, kRouteScanned><<<blocks, kRouteThreads, 0, st>>>(ids, n, num_experts, bits, counts, totals, blocks, row_of_slot, slot_of_row, offsets);
}

// What dispatch, combine and its backward pass have in common; null pointers that a call does not use are its own affair.
const char* check_move(int dtype, int64_t tokens, int topk, int64_t dim, const int32_t* row_of_slot, const void* weights, int weight_dtype) {
    if (!known_dtype(dtype)) return "unknown dtype";
    if (tokens < 0) return "tokens is negative";
    if (topk < 1 || topk > SAR_MAX_TOPK) return "topk must be 1 to 64";
    if (tokens > INT32_MAX / topk) return "tokens * topk must stay below 2^31";
    if (dim < 1 || dim > (1 << 24)) return "dim must be 1 to 2^24";
    if (weights && weight_dtype != SAR_F32 && weight_dtype != dtype) return "weights must be of dtype or 32-bit floats";
    if (weights && !aligned(weights, elem_size(weight_dtype))) return "weights are not aligned to their element size";
    if (tokens && (!row_of_slot || !aligned(row_of_slot, 4))) return "row_of_slot is null or not aligned";
    return nullptr;
}

MoveArgs move_args(int dtype, int64_t tokens, int topk, int64_t dim, const int32_t* row_of_slot, const void* weights, int weight_dtype) {
    MoveArgs a{};
    a.weights = (const char*)weights;
    a.row_of_slot = row_of_slot;
    a.tokens = (uint64_t)tokens;
    a.topk = (uint32_t)topk;
    a.nrows = (uint32_t)(tokens * topk);
    a.dim = (uint32_t)dim;
    const uint32_t ve = (uint32_t)dim < 16u / elem_size(dtype) ? 1u : 16u / elem_size(dtype);
    a.nvec = (a.dim + ve - 1) / ve;
    a.row_bytes = a.dim * elem_size(dtype);
    a.weights_f32 = weight_dtype == SAR_F32;
    return a;
}

// Calls that move this much and more stream their rows past the caches: what does not fit into the 256 MB Infinity
// Cache only pushes out what does, and a cached store's way to memory is paid for by the next call.  Measured, cached
// against streaming, as a chain with a pass over the result behind it: dispatch of 537 MB 407 against 381 us (chain
// with its combine), of 268 MB 173 against 184; eight partials of 8192 x 4096 (1.2 GB) 432 against 397, of 4096 222
// against 213, of 2048 (302 MB) 107 against 118.  The streams that come once beside eight others stay cached all the same:
// dispatch's tokens (230 -> 212 us with its gradient), the residual and hidden of reduce_norm (221 -> 205), its total for the
// backward pass (287 -> 272).
constexpr uint64_t kStreamBytes = 512ull << 20;

// calls f(integral_constant<bool, B>)
template <class F> void with_bool(bool b, F&& f) {
    if (b) f(std::true_type{});
    else f(std::false_type{});
}

// One vector a lane: two and four were level for the large calls (16384 tokens of 2048, eight choices: combine 101 us with
// two, 101 with one; dispatch with its gradient 212 with four, 219 with two, 210 with one) and slower for the small ones (32
// tokens: 3.9 us with four, 3.1) and for rows that do not fill them (3000 of 7168: 73 with four, 64).
dim3 move_grid(const MoveArgs& a) {
    const uint64_t groups = (a.tokens + kMoveWaves - 1) / kMoveWaves;
    return dim3((a.nvec + kWave - 1) / kWave, (uint32_t)std::min<uint64_t>(groups, 65535u));
}

// calls f(integral_constant<int, VE>, integral_constant<bool, NT>) for a call
template <int DT, class F> void with_move_shape(const MoveArgs& a, F&& f) {
    if (a.dim < kVec<DT>) f(std::integral_constant<int, 1>{}, std::false_type{});
    else with_bool(((uint64_t)a.nrows + a.tokens) * a.row_bytes >= kStreamBytes, [&](auto nt) { f(std::integral_constant<int, kVec<DT>>{}, nt); });
}

template <int DT> void launch_dispatch(hipStream_t st, const MoveArgs& a) {
    with_bool(a.weights != nullptr, [&](auto weighted) {
        with_move_shape<DT>(a, [&](auto ve, auto nt) {
            dispatch_kernel<DT, decltype(ve)::value, decltype(nt)::value, decltype(weighted)::value><<<move_grid(a), kMoveThreads, 0, st>>>(a);
        });
    });
}

template <int DT> void launch_combine(hipStream_t st, const MoveArgs& a) {
    with_move_shape<DT>(a, [&](auto ve, auto nt) { combine_kernel<DT, decltype(ve)::value, decltype(nt)::value><<<move_grid(a), kMoveThreads, 0, st>>>(a); });
}

// A wave takes a token, with as many vectors a lane as the row has; four waves share one where the row is longer than
// that, or where there are too few tokens to keep the chip busy (32 tokens of 2048, eight choices: 5.4 us shared, 7.3 not;
// 4099 of 1001, two choices: 13.3 shared, 11.7 not; nothing in between was measured).  Two rows at a time: four cost registers and with them waves (50000
// tokens of 256, one choice: 36.7 us against 46.1).
template <int DT> void launch_combine_backward(hipStream_t st, const MoveArgs& a) {
    const bool shared = a.nvec > 4 * kWave || (a.nvec > kWave && a.tokens < 2048);
    const uint64_t groups = shared ? a.tokens : (a.tokens + kMoveWaves - 1) / kMoveWaves;
    const uint32_t grid = (uint32_t)std::min<uint64_t>(groups, 1u << 20);
    const bool nt = ((uint64_t)a.nrows * (a.out ? 2 : 1) + a.tokens) * a.row_bytes >= kStreamBytes;
    if (a.dim < kVec<DT>) {
        combine_backward_kernel<DT, 1, 1, 1, false><<<grid, kMoveThreads, 0, st>>>(a);
        return;
    }
    with_bool(nt, [&](auto stream) {
        constexpr bool NT = decltype(stream)::value;
        if (shared) combine_backward_kernel<DT, kVec<DT>, 2, 4, NT><<<grid, kMoveThreads, 0, st>>>(a);
        else if (a.nvec <= kWave) combine_backward_kernel<DT, kVec<DT>, 1, 1, NT><<<grid, kMoveThreads, 0, st>>>(a);
        else if (a.nvec <= 2 * kWave) combine_backward_kernel<DT, kVec<DT>, 2, 1, NT><<<grid, kMoveThreads, 0, st>>>(a);
        else combine_backward_kernel<DT, kVec<DT>, 4, 1, NT><<<grid, kMoveThreads, 0, st>>>(a);
    });
}

// Threads and vectors per thread for a row: one vector a thread as far as 1024 threads reach.
struct NormShape { uint32_t threads; int vectors; bool single; };
NormShape norm_shape(int dtype, int64_t dim) {
    const uint32_t ve = 16u / elem_size(dtype);
    if ((uint32_t)dim < ve) return {kWave, 1, true};
    const uint32_t nvec = ((uint32_t)dim + ve - 1) / ve;
    const int v = nvec <= 1024 ? 1 : nvec <= 2048 ? 2 : 4;
    const uint32_t threads = ((nvec + v - 1) / v + kWave - 1) / kWave * kWave;
    return {threads, v, false};
}

// Tokens a workgroup of the backward pass has in hand.
uint32_t norm_backward_rows(const NormShape& s) { return s.vectors > 1 || s.threads > kRowsThreads ? 1u : kRowsThreads / s.threads; }

// Workgroups of the backward pass: as many as the chip holds at once (a token for each row of threads is enough: 8 tokens
// of 4096 take 9.6 us so, 13.1 with two tokens in turn and fewer column sums, 20.3 with four; 1537 of 1001 15.0, 15.2, 19.4).
uint32_t norm_backward_groups(int64_t tokens, int64_t dim, int dtype) {
    const NormShape s = norm_shape(dtype, dim);
    const uint32_t rows = norm_backward_rows(s);
    const uint64_t resident = 256u * std::max(1u, 1024u / (s.threads * rows));
    return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(resident, ((uint64_t)tokens + rows - 1) / rows));
}

const char* check_norm(const sar_reduce_norm_args* a) {
    if (!a) return "the argument struct is null";
    if (!known_dtype(a->dtype)) return "unknown dtype";
    if (a->tokens < 0) return "tokens is negative";
    if (a->dim < 1 || a->dim > SAR_MAX_NORM_DIM) return "dim must be 1 to 16384";
    if (a->tokens > (int64_t)1 << 40) return "too many tokens";
    if (a->sources < 1 || a->sources > SAR_MAX_RANKS) return "sources must be 1 to 64";
    if (a->copies < 1 || a->copies > SAR_MAX_RANKS) return "copies must be 1 to 64";
    if (!(a->eps >= 0.f) || a->eps > 3.4e38f) return "eps must be a number, zero or more";
    if (a->pre_weight && a->pre_dtype != a->dtype && a->pre_dtype != SAR_F32) return "pre_weight must be of dtype or 32-bit floats";
    if (a->post_weight && a->post_dtype != a->dtype && a->post_dtype != SAR_F32) return "post_weight must be of dtype or 32-bit floats";
    if (a->gate_kind < SAR_GATE_NONE || a->gate_kind > SAR_GATE_FULL) return "unknown gate kind";
    if (a->gate_kind != SAR_GATE_NONE && !a->gate && a->tokens) return "gate is null";
    if (a->gate_kind != SAR_GATE_NONE && a->gate_dtype != a->dtype && a->gate_dtype != SAR_F32) return "gate must be of dtype or 32-bit floats";
    const uint64_t es = elem_size(a->dtype);
    if (!aligned(a->residual, es) || !aligned(a->pre_weight, a->pre_weight ? elem_size(a->pre_dtype) : 1) ||
        !aligned(a->post_weight, a->post_weight ? elem_size(a->post_dtype) : 1) || !aligned(a->gate, a->gate_kind ? elem_size(a->gate_dtype) : 1))
        return "a pointer is not aligned to its element size";
    if (a->tokens && !a->residual) return "residual is null";
    return nullptr;
}

NormArgs norm_args(const sar_reduce_norm_args* a) {
    NormArgs k{};
    k.residual = (const char*)a->residual;
    k.pre = (const char*)a->pre_weight;
    k.post = (const char*)a->post_weight;
    k.gate = (const char*)a->gate;
    k.hidden = (char*)a->hidden;
    k.normed = (char*)a->normed;
    k.total = a->total;
    k.stats = a->stats;
    k.tokens = (uint64_t)a->tokens;
    k.dim = (uint32_t)a->dim;
    const uint32_t es = elem_size(a->dtype), ve = a->dim < 16 / es ? 1u : 16u / es;
    k.nvec = (k.dim + ve - 1) / ve;
    k.row_bytes = k.dim * es;
    k.copy_bytes = k.tokens * k.row_bytes;
    k.sources = (uint32_t)a->sources;
    k.copies = (uint32_t)a->copies;
    k.gate_kind = (uint32_t)a->gate_kind;
    k.pre_f32 = a->pre_dtype == SAR_F32;
    k.post_f32 = a->post_dtype == SAR_F32;
    k.gate_f32 = a->gate_dtype == SAR_F32;
    k.eps = a->eps;
    k.residual_scale = a->residual_scale;
    k.inv_dim = 1.f / (float)a->dim;
    return k;
}

// calls f(integral_constant<int, VE>, integral_constant<int, V>) for a shape
template <int DT, class F> void with_norm_shape(const NormShape& s, F&& f) {
    using std::integral_constant;
    if (s.single) f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (s.vectors == 1) f(integral_constant<int, kVec<DT>>{}, integral_constant<int, 1>{});
    else if (s.vectors == 2) f(integral_constant<int, kVec<DT>>{}, integral_constant<int, 2>{});
    else if constexpr (DT == SAR_F32) f(integral_constant<int, kVec<DT>>{}, integral_constant<int, 4>{});
}

template <int DT> void launch_norm(hipStream_t st, const NormArgs& a, const NormShape& s) {
    const uint32_t grid = (uint32_t)std::min<uint64_t>(a.tokens, 1u << 20);
    const uint64_t rows = a.sources + 2 + (a.normed ? a.copies : 0) + (a.total ? 4 / ElemSize<DT>::value : 0);
    with_bool(rows * a.copy_bytes >= kStreamBytes, [&](auto nt) {
        // a finished output asks for no batch of rows: fewer registers, more rows in flight (4096 of 4096: 30.1 -> 25.9 us)
        with_bool(a.sources == 1, [&](auto one) {
            with_norm_shape<DT>(s, [&](auto ve, auto v) { reduce_norm_kernel<DT, decltype(ve)::value, decltype(v)::value, decltype(one)::value, decltype(nt)::value><<<grid, s.threads, 0, st>>>(a); });
        });
    });
}

template <int DT> void launch_norm_backward(hipStream_t st, const NormBackwardArgs& b, const NormShape& s, uint32_t grid) {
    const NormArgs& a = b.f;
    const uint64_t rows = (b.grad_partials ? a.sources : 0) + 3 + (b.grad_normed ? a.copies : 0) + (b.total_f32 ? 4 / ElemSize<DT>::value : 1);
    with_bool(rows * a.copy_bytes >= kStreamBytes, [&](auto nt) {
        with_bool(a.sources == 1 && a.copies == 1, [&](auto one) {
            with_norm_shape<DT>(s, [&](auto ve, auto v) {
                constexpr int VE = decltype(ve)::value, V = decltype(v)::value;
                constexpr bool ONE = decltype(one)::value && V == 1;
                reduce_norm_backward_kernel<DT, VE, V, ONE, decltype(nt)::value><<<grid, s.threads * norm_backward_rows(s), 0, st>>>(b);
            });
        });
    });
}

}  // namespace
}  // namespace sar

using namespace sar;

extern "C" {

uint64_t sar_route_workspace(int64_t tokens, int topk, int num_experts) {
    if (tokens < 0 || topk < 1 || topk > SAR_MAX_TOPK || num_experts < 1 || num_experts > SAR_MAX_EXPERTS || tokens > INT32_MAX / topk) return 0;
    const uint64_t n = (uint64_t)tokens * (uint64_t)topk;
    return n <= kRouteOne ? 0 : (route_blocks(n) + 1) * (uint64_t)num_experts * 4u;
}

int sar_route(int device, void* stream, const void* experts, int index_bytes, int64_t tokens, int topk, int num_experts,
              int32_t* row_of_slot, int32_t* slot_of_row, int32_t* offsets, void* workspace, uint64_t workspace_bytes) {
    return guarded([&]() -> int {
        if (index_bytes != 4 && index_bytes != 8) return refuse("index_bytes must be 4 or 8");
        if (tokens < 0) return refuse("tokens is negative");
        if (topk < 1 || topk > SAR_MAX_TOPK) return refuse("topk must be 1 to 64");
        if (num_experts < 1 || num_experts > SAR_MAX_EXPERTS) return refuse("num_experts must be 1 to 1024");
        if (tokens > INT32_MAX / topk) return refuse("tokens * topk must stay below 2^31");
        if (!offsets || !aligned(offsets, 4)) return refuse("offsets is null or not aligned");
        if (tokens && (!experts || !row_of_slot || !slot_of_row)) return refuse("a pointer is null");
        if (!aligned(experts, (uint64_t)index_bytes) || !aligned(row_of_slot, 4) || !aligned(slot_of_row, 4)) return refuse("a pointer is not aligned to its element size");
        const uint64_t need = sar_route_workspace(tokens, topk, num_experts);
        if (need && (!workspace || !aligned(workspace, 4) || workspace_bytes < need)) return refuse("the workspace is smaller than sar_route_workspace()");
        OnDevice on(device);
        if (on.error() != hipSuccess) return not_current(device, on.error());
        const uint32_t n = (uint32_t)(tokens * topk);
        if (index_bytes == 8) launch_route<int64_t>((hipStream_t)stream, experts, n, (uint32_t)num_experts, row_of_slot, slot_of_row, offsets, (uint32_t*)workspace);
        else launch_route<int32_t>((hipStream_t)stream, experts, n, (uint32_t)num_experts, row_of_slot, slot_of_row, offsets, (uint32_t*)workspace);
        return launched("sar_route");
    });
}

int sar_dispatch(int device, void* stream, int dtype, const void* token_rows, int64_t tokens, int topk, int64_t dim,
                 const int32_t* row_of_slot, const int32_t* offsets, int num_experts, const void* weights, int weight_dtype,
                 void* rows) {
    return guarded([&]() -> int {
        if (const char* why = check_move(dtype, tokens, topk, dim, row_of_slot, weights, weight_dtype)) return refuse(why);
        if (num_experts < 1 || num_experts > SAR_MAX_EXPERTS) return refuse("num_experts must be 1 to 1024");
        if (tokens == 0) return SAR_OK;
        if (!token_rows || !rows || !offsets) return refuse("a pointer is null");
        if (!aligned(token_rows, elem_size(dtype)) || !aligned(rows, elem_size(dtype)) || !aligned(offsets, 4)) return refuse("a pointer is not aligned to its element size");
        OnDevice on(device);
        if (on.error() != hipSuccess) return not_current(device, on.error());
        MoveArgs a = move_args(dtype, tokens, topk, dim, row_of_slot, weights, weight_dtype);
        a.in = (const char*)token_rows;
        a.out = (char*)rows;
        a.total = offsets + num_experts;
        with_dtype(dtype, [&](auto dt) { launch_dispatch<decltype(dt)::value>((hipStream_t)stream, a); });
        return launched("sar_dispatch");
    });
}

int sar_combine(int device, void* stream, int dtype, const void* rows, int64_t tokens, int topk, int64_t dim,
                const int32_t* row_of_slot, const void* weights, int weight_dtype, void* out) {
    return guarded([&]() -> int {
        if (const char* why = check_move(dtype, tokens, topk, dim, row_of_slot, weights, weight_dtype)) return refuse(why);
        if (tokens == 0) return SAR_OK;
        if (!rows || !out) return refuse("a pointer is null");
        if (!aligned(rows, elem_size(dtype)) || !aligned(out, elem_size(dtype))) return refuse("a pointer is not aligned to its element size");
        OnDevice on(device);
        if (on.error() != hipSuccess) return not_current(device, on.error());
        MoveArgs a = move_args(dtype, tokens, topk, dim, row_of_slot, weights, weight_dtype);
        a.in = (const char*)rows;
        a.out = (char*)out;
        with_dtype(dtype, [&](auto dt) { launch_combine<decltype(dt)::value>((hipStream_t)stream, a); });
        return launched("sar_combine");
    });
}

int sar_combine_backward(int device, void* stream, int dtype, const void* grad, const void* rows, int64_t tokens, int topk,
                         int64_t dim, const int32_t* row_of_slot, const int32_t* offsets, int num_experts,
                         const void* weights, int weight_dtype, void* grad_rows, void* grad_weights) {
    return guarded([&]() -> int {
        if (const char* why = check_move(dtype, tokens, topk, dim, row_of_slot, weights, weight_dtype)) return refuse(why);
        if (num_experts < 1 || num_experts > SAR_MAX_EXPERTS) return refuse("num_experts must be 1 to 1024");
        if (tokens == 0) return SAR_OK;
        if (!grad || !rows || !weights || !grad_weights || (grad_rows && !offsets)) return refuse("a pointer is null");
        const uint64_t es = elem_size(dtype);
        if (!aligned(grad, es) || !aligned(rows, es) || !aligned(grad_rows, es) || !aligned(offsets, 4) || !aligned(grad_weights, elem_size(weight_dtype)))
            return refuse("a pointer is not aligned to its element size");
        OnDevice on(device);
        if (on.error() != hipSuccess) return not_current(device, on.error());
        MoveArgs a = move_args(dtype, tokens, topk, dim, row_of_slot, weights, weight_dtype);
        a.in = (const char*)grad;
        a.rows = (const char*)rows;
        a.out = (char*)grad_rows;
        a.grad_weights = (char*)grad_weights;
        a.total = offsets ? offsets + num_experts : nullptr;
        with_dtype(dtype, [&](auto dt) { launch_combine_backward<decltype(dt)::value>((hipStream_t)stream, a); });
        return launched("sar_combine_backward");
    });
}

int sar_reduce_norm(int device, void* stream, const sar_reduce_norm_args* args) {
    return guarded([&]() -> int {
        if (const char* why = check_norm(args)) return refuse(why);
        if (args->tokens == 0) return SAR_OK;
        if (!args->partials) return refuse("the list of partials is null");
        const uint64_t es = elem_size(args->dtype);
        for (int s = 0; s < args->sources; ++s)
            if (!args->partials[s] || !aligned(args->partials[s], es)) return refuse("a partial is null or not aligned to its element size");
        if ((args->pre_weight != nullptr) != (args->normed != nullptr)) return refuse("pre_weight and normed go together");
        if (!aligned(args->hidden, es) || !aligned(args->normed, es) || !aligned(args->total, 4) || !aligned(args->stats, 4))
            return refuse("a pointer is not aligned to its element size");
        OnDevice on(device);
        if (on.error() != hipSuccess) return not_current(device, on.error());
        NormArgs a = norm_args(args);
        for (int s = 0; s < args->sources; ++s) a.partials[s] = (const char*)args->partials[s];
        const NormShape shape = norm_shape(args->dtype, args->dim);
        with_dtype(args->dtype, [&](auto dt) { launch_norm<decltype(dt)::value>((hipStream_t)stream, a, shape); });
        return launched("sar_reduce_norm");
    });
}

uint64_t sar_reduce_norm_workspace(int64_t tokens, int64_t dim, int dtype) {
    if (tokens < 0 || dim < 1 || dim > SAR_MAX_NORM_DIM || !known_dtype(dtype)) return 0;
    const uint64_t groups = norm_backward_groups(tokens, dim, dtype);
    return groups == 1 ? 0 : groups * 3u * (uint64_t)dim * 4u;
}

int sar_reduce_norm_backward(int device, void* stream, const sar_reduce_norm_args* forward, const sar_reduce_norm_grads* g) {
    return guarded([&]() -> int {
        if (const char* why = check_norm(forward)) return refuse(why);
        if (!g) return refuse("the struct of gradients is null");
        const uint64_t es = elem_size(forward->dtype);
        const bool channel = forward->gate_kind == SAR_GATE_CHANNEL;
        if (g->grad_normed && !forward->pre_weight) return refuse("grad_normed without pre_weight");
        if (g->grad_pre_weight && !forward->pre_weight) return refuse("grad_pre_weight without pre_weight");
        if (g->grad_post_weight && !forward->post_weight) return refuse("grad_post_weight without post_weight");
        if (g->grad_gate && forward->gate_kind == SAR_GATE_NONE) return refuse("grad_gate without a gate");
        // with no tokens the kernel still runs, for the weights' zero gradients, and holds a channel gate in registers
        if (channel && !forward->gate) return refuse("gate is null");
        if (g->total_dtype != SAR_F32 && g->total_dtype != forward->dtype) return refuse("total must be of dtype or 32-bit floats");
        if (forward->tokens && (!g->total || !forward->stats)) return refuse("total or stats is null");
        if (!aligned(g->total, elem_size(g->total_dtype)) || !aligned(forward->stats, 4) || !aligned(g->grad_hidden, es) || !aligned(g->grad_normed, es) ||
            !aligned(g->grad_partials, es) || !aligned(g->grad_residual, es) ||
            !aligned(g->grad_pre_weight, g->grad_pre_weight ? elem_size(forward->pre_dtype) : 1) ||
            !aligned(g->grad_post_weight, g->grad_post_weight ? elem_size(forward->post_dtype) : 1) ||
            !aligned(g->grad_gate, g->grad_gate ? elem_size(forward->gate_dtype) : 1))
            return refuse("a pointer is not aligned to its element size");
        const uint64_t need = sar_reduce_norm_workspace(forward->tokens, forward->dim, forward->dtype);
        if (need && (!g->workspace || !aligned(g->workspace, 4) || g->workspace_bytes < need))
            return refuse("the workspace is smaller than sar_reduce_norm_workspace()");
        OnDevice on(device);
        if (on.error() != hipSuccess) return not_current(device, on.error());
        NormBackwardArgs b{};
        b.f = norm_args(forward);
        b.total = (const char*)g->total;
        b.total_f32 = g->total_dtype == SAR_F32;
        b.grad_hidden = (const char*)g->grad_hidden;
        b.grad_normed = (const char*)g->grad_normed;
        b.grad_partials = (char*)g->grad_partials;
        b.grad_residual = (char*)g->grad_residual;
        b.grad_gate = channel ? nullptr : (char*)g->grad_gate;
        b.columns = (float*)g->workspace;
        b.grad_weights[0] = (char*)g->grad_pre_weight;
        b.grad_weights[1] = (char*)g->grad_post_weight;
        b.grad_weights[2] = channel ? (char*)g->grad_gate : nullptr;
        b.weights_f32[0] = b.f.pre_f32;
        b.weights_f32[1] = b.f.post_f32;
        b.weights_f32[2] = b.f.gate_f32;
        const uint32_t groups = norm_backward_groups(forward->tokens, forward->dim, forward->dtype);
        const NormShape shape = norm_shape(forward->dtype, forward->dim);
        b.row_threads = shape.threads;
        with_dtype(forward->dtype, [&](auto dt) { launch_norm_backward<decltype(dt)::value>((hipStream_t)stream, b, shape, groups); });
        if (int rc = launched("sar_reduce_norm_backward")) return rc;
        if (groups > 1 && (b.grad_weights[0] || b.grad_weights[1] || b.grad_weights[2])) {
            ColumnArgs c{};
            c.columns = b.columns;
            for (int i = 0; i < 3; ++i) { c.out[i] = b.grad_weights[i]; c.f32[i] = b.weights_f32[i]; }
            c.rows = groups;
            c.dim = b.f.dim;
            const dim3 grid((c.dim + 31u) / 32u, 3);
            with_dtype(forward->dtype, [&](auto dt) { column_sum_kernel<decltype(dt)::value><<<grid, 1024, 0, (hipStream_t)stream>>>(c); });
            return launched("sar_reduce_norm_backward");
        }
        return SAR_OK;
    });
}

}  // extern "C"
