// Selection of a router row's experts without k rounds over the row.
#pragma once
#include "qmoe_int8.hpp"

namespace qmoe {

// The k largest of a row held NV values a lane, as RouterRow::select picks them (descending, NaN last, lower id on ties):
// lane s gets selection s.
template <int NV> struct RowIds {
    float v[NV];
    __device__ __forceinline__ void load(const float* z, int n) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = ldg<float>(z + (lane + 64 * j < n ? lane + 64 * j : 0));
    }
    // The k-th largest of the lanes' largest keys is a bound that at least k keys reach, and hardly more: those are gathered,
    // one a lane, and ranked.  (k rounds of "largest of the wave, take it out" cost 4.5 us for ten of 512, this one fifth.)
    // More than 64 keys reach the bound only where many are equal: then the rounds.  `scratch`: 64 entries of this wave.
    __device__ __forceinline__ int select(int n, int k, uint2* scratch) {
        const int lane = threadIdx.x & 63;
        uint32_t key[NV], top = 0u;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const uint32_t o = order_key(v[j]);
            key[j] = lane + 64 * j < n ? (o ? o : 1u) : 0u;
            top = key[j] > top ? key[j] : top;
        }
        int ahead = 0;
#pragma unroll
        for (int i = 0; i < 64; ++i) ahead += (uint32_t)__builtin_amdgcn_readlane((int)top, i) > top;
        uint32_t bound = ~wave_max_u32(ahead < k ? ~top : 0u);
        bound = bound ? bound : 1u;
        int count = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const bool in = key[j] >= bound;
            const unsigned long long m = __ballot(in);
            const int at = count + __popcll(m & ((1ull << lane) - 1));
            if (in && at < 64) scratch[at] = make_uint2(key[j], (uint32_t)(lane + 64 * j));
            count += __popcll(m);
        }
        if (__builtin_expect(count > 64, 0)) return rounds(key, k);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
        // (gathered in ascending id: among equal keys the lower lane comes first)
        const uint2 mine = lane < count ? scratch[lane] : make_uint2(0u, 0u);
        int rank = 0;
        for (int i = 0; i < count; ++i) {
            const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)mine.x, i);
            rank += other > mine.x || (other == mine.x && i < lane);
        }
        return __builtin_amdgcn_ds_permute((lane < count ? rank : lane) * 4, (int)mine.y);
    }
    // Ids and weights of the row z (held in v): the formulas of RouterRow::select, with the selection above.
    __device__ __forceinline__ void route(const float* z, int n, int k, float floor_value, int renorm, uint2* scratch, float& weight, int64_t& id) {
        const int lane = threadIdx.x & 63;
        uint32_t best = 0u;
        bool nan = false;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const uint32_t o = lane + 64 * j < n ? order_key(v[j]) : 1u;
            nan |= o == 0u;
            best = o > best ? o : best;
        }
        const float m = __any(nan) ? __uint_as_float(0x7FC00000u) : key_value(wave_max_u32(best));
        double part = 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (lane + 64 * j < n) part += (double)expf(v[j] - m);
        const float denom = (float)wave_sum_f64(part);
        const int mine = select(n, k, scratch);
        const float p = lane < k ? expf(ldg<float>(z + mine) - m) / denom : 0.0f;
        float mass = 0.0f;
        for (int slot = 0; slot < k; ++slot) mass += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), slot));
        weight = renorm ? p / (isnan(mass) ? mass : fmaxf(mass, floor_value)) : p;
        id = mine;
    }
    __device__ __forceinline__ static int rounds(uint32_t (&key)[NV], int k) {
        const int lane = threadIdx.x & 63;
        int mine = 0;
        for (int slot = 0; slot < k; ++slot) {
            uint32_t c = 0u;
#pragma unroll
            for (int j = 0; j < NV; ++j) c = key[j] > c ? key[j] : c;
            const uint32_t win = wave_max_u32(c);
            int wj = 0;
            unsigned long long holders = 0ull;
#pragma unroll
            for (int j = NV - 1; j >= 0; --j) {
                const unsigned long long b = __ballot(key[j] == win);
                if (b) { wj = j; holders = b; }
            }
            const int wl = __builtin_ctzll(holders);
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (j == wj) key[j] = lane == wl ? 0u : key[j];
            if (lane == slot) mine = wl + 64 * wj;
        }
        return mine;
    }
};

}  // namespace qmoe
