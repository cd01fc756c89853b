// paged_ops.hip -- a serving step over a paged cache, around its attention
// (paged_attn.hip): the plan of the step, the rotary step with the write into
// the pages, and the rules on the logits.  No counterpart in the reference,
// which runs one sequence.  What each computes is declared in the header.
#include <hip/hip_fp16.h>

#include <climits>
#include <cmath>

#include "paged_common.h"
#include "qk_common.h"

namespace rf {

// ---- the plan ----------------------------------------------------------------------------
//
// Two prefix sums over the requests (rows, then pages of those whose rows and
// table fit), the new pages off the stack, then one position and one slot a
// row.  Bound by latency: a request is two ints and a row two more (57 KB of
// output at 14 k rows).  One workgroup scans; where there are few rows it
// writes them as well (one launch), else a second launch spreads them over
// the chip.  64 requests of one token 5.7 us; 300 of 14 k rows 5.4 and 3.8.

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

// Inclusive prefix sum over the workgroup; total: of all its values.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* wave_sums, int64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();                             // the last scan's readers are done
    if (lane == 63) wave_sums[wave] = v;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int w = 0; w < kPlanWaves; ++w) {
        const int64_t s = wave_sums[w];
        if (w < wave) before += s;
        all += s;
    }
    *total = all;
    return before + v;
}

// (page sizes are powers of two)
__device__ __forceinline__ int64_t pages_for(int64_t n, int page) { return (n + page - 1) >> (__ffs(page) - 1); }

// Position and slot of row r, whose request is the last one that starts at or
// before it (requests of no rows share their start with the next).  starts: q_start,
// in LDS where there is room for it.
__device__ __forceinline__ void plan_row(const rf_paged_plan& p, const int* starts, int r) {
    int lo = 0, hi = p.num_seqs;                 // starts[lo] <= r; r < starts[hi] unless r is padding
    if (r < starts[hi]) {
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (starts[mid] <= r)
                lo = mid;
            else
                hi = mid;
        }
        const int n = p.new_lens[lo], kv = p.kv_lens[lo];
        if (kv > 0) {
            const int pos = kv - n + (r - starts[lo]), sh = __ffs(p.page_size) - 1;
            p.positions[r] = pos;
            // (an entry that names no page may lie anywhere: in 32 bits its slot could be another page's)
            const int64_t slot = (int64_t)p.block_tables[(int64_t)lo * p.max_blocks + (pos >> sh)] * p.page_size +
                                 (pos & (p.page_size - 1));
            p.slots[r] = slot == (int)slot ? (int)slot : -1;
            return;
        }
    }
    p.positions[r] = 0;
    p.slots[r] = -1;
}

// ROWS: writes the rows too (then there are at most kPlanThreads requests).
template <bool ROWS>
__global__ __launch_bounds__(kPlanThreads) void rf_paged_plan_kernel(const rf_paged_plan p) {
    __shared__ int64_t sums[kPlanWaves];
    __shared__ int64_t page_end[kPlanThreads];   // pages asked for up to and with request b0 + t
    __shared__ int page_first[kPlanThreads];     // its first new column
    __shared__ int starts[ROWS ? kPlanThreads + 1 : 1];
    __shared__ int granted_end;                  // pages of the granted requests so far: a prefix of those asked for
    const int t = threadIdx.x;
    const int64_t n_free = min(max(p.free_in[0], 0), p.num_pages);
    int64_t rows_before = 0, pages_before = 0;
    if (t == 0) {
        p.q_start[0] = 0;
        starts[0] = 0;
        granted_end = 0;
    }
    for (int b0 = 0; b0 < p.num_seqs; b0 += kPlanThreads) {
        const int b = b0 + t;
        const bool there = b < p.num_seqs;
        const int64_t n = there ? p.new_lens[b] : 0, ctx = there ? p.ctx_in[b] : 0;
        int64_t rows, pages;
        const int64_t row_end = rows_before + block_scan(n > 0 ? n : 0, sums, &rows);
        const int64_t have = pages_for(ctx, p.page_size), want = pages_for(ctx + n, p.page_size);
        const bool fits = there && n >= 0 && ctx >= 0 && row_end <= p.max_rows && want <= p.max_blocks &&
                          ctx + n <= INT_MAX;
        const int64_t need = fits ? want - have : 0;
        const int64_t end = pages_before + block_scan(need, sums, &pages);
        const bool granted = fits && (need == 0 || end <= n_free);
        if (there) {
            const int start = (int)min(row_end, (int64_t)p.max_rows);
            p.q_start[b + 1] = start;
            if constexpr (ROWS) starts[t + 1] = start;
            p.kv_lens[b] = granted ? (int)(ctx + n) : 0;
            p.ctx_out[b] = granted ? (int)(ctx + n) : (int)ctx;
        }
        page_end[t] = end;
        page_first[t] = (int)have;
        if (granted && need > 0) atomicMax(&granted_end, (int)end);
        __syncthreads();
        // page i belongs to the first of these requests whose end passes it
        for (int64_t i = pages_before + t; i < granted_end; i += kPlanThreads) {
            int lo = 0, hi = kPlanThreads - 1;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (page_end[mid] > i)
                    hi = mid;
                else
                    lo = mid + 1;
            }
            const int64_t begin = lo > 0 ? page_end[lo - 1] : pages_before;
            p.block_tables[(int64_t)(b0 + lo) * p.max_blocks + page_first[lo] + (i - begin)] =
                p.free_pages[n_free - 1 - i];
        }
        rows_before += rows;
        pages_before += pages;
        __syncthreads();                         // page_end is read no more
    }
    __syncthreads();                             // (no requests: granted_end)
    if (t == 0) p.free_out[0] = (int)(n_free - granted_end);
    if constexpr (ROWS)                          // this workgroup's own global writes, read back behind the barrier
        for (int r = t; r < p.max_rows; r += kPlanThreads) plan_row(p, starts, r);
}

constexpr int kStartsInLds = 4096;

__global__ __launch_bounds__(256) void rf_paged_rows_kernel(const rf_paged_plan p) {
    __shared__ int starts[kStartsInLds];
    const int r = blockIdx.x * 256 + threadIdx.x;
    if (p.num_seqs < kStartsInLds) {
        for (int i = threadIdx.x; i <= p.num_seqs; i += 256) starts[i] = p.q_start[i];
        __syncthreads();
        if (r < p.max_rows) plan_row(p, starts, r);
    } else if (r < p.max_rows) {
        plan_row(p, p.q_start, r);
    }
}

// The pages of ended requests, one workgroup: a scan over the requests, then each of the
// 16 waves copies those of its 64 one request after the other.  Bound by those copies'
// latency: one request of 640 positions (40 pages) 3.7 us, 64 of 2000 23.6, one of 100,000 14.6.
__global__ __launch_bounds__(kPlanThreads) void rf_paged_release_kernel(const int* __restrict__ ended, int* ctx_lens,
                                                                        const int* __restrict__ tables,
                                                                        int* free_pages, int* free_count, int num_seqs,
                                                                        int max_blocks, int page, int num_pages) {
    __shared__ int64_t sums[kPlanWaves];
    const int t = threadIdx.x, lane = t & 63;
    const int64_t n_free = min(max(free_count[0], 0), num_pages);
    int64_t before = n_free, top = n_free;
    for (int b0 = 0; b0 < num_seqs; b0 += kPlanThreads) {
        const int b = b0 + t;
        const int64_t ctx = b < num_seqs && ended[b] != 0 ? max(ctx_lens[b], 0) : 0;
        int64_t n = pages_for(ctx, page), all;
        if (n > max_blocks) n = 0;
        const int64_t end = before + block_scan(n, sums, &all);
        const bool back = n > 0 && end <= num_pages;
        if (back) ctx_lens[b] = 0;
        // a wave copies its requests' pages one request after the other
        uint64_t left = __ballot(back);
        while (left) {
            const int l = __builtin_ctzll(left);
            left &= left - 1;
            const int64_t k = __shfl(n, l), at = __shfl(end, l) - k;
            const int* row = tables + (int64_t)(b0 + (t & ~63) + l) * max_blocks;
            for (int64_t i = lane; i < k; i += 64) free_pages[at + i] = row[i];
        }
        // handed back are a prefix of the ones that ask: the top is the last such end
        int64_t unused = back ? end : 0;
#pragma unroll
        for (int o = 32; o; o >>= 1) unused = max(unused, (int64_t)__shfl_xor(unused, o));
        __syncthreads();
        if (lane == 0) sums[t >> 6] = unused;
        __syncthreads();
        for (int w = 0; w < kPlanWaves; ++w) top = max(top, sums[w]);
        before += all;
    }
    __syncthreads();
    if (t == 0) free_count[0] = (int)top;
}

// ---- the rotary step into the pages --------------------------------------------------------
//
// theta_i / 2 pi: positions times this, less whole turns, is the angle to 2^-53
// of the position's turns, and then rounded to fp32: off by up to 2^-26 of a turn, 2^-23
// of a radian, at any position -- at 130,000 an angle held in fp32 throughout is off
// by up to 2^-8.
__global__ void rf_rope_turns_kernel(double* __restrict__ turns, int rot, double base, int mode, double factor,
                                     double lo, double hi, const float* __restrict__ freq_scale) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= rot / 2) return;
    double theta = pow(base, -2.0 * i / rot);
    if (freq_scale != nullptr) theta /= (double)freq_scale[i];
    if (mode == RF_ROPE_LINEAR) theta /= factor;
    if (mode == RF_ROPE_YARN) {
        const double r = fmin(fmax((i - lo) / fmax(hi - lo, 0.001), 0.0), 1.0);
        theta = theta / factor * r + theta * (1.0 - r);
    }
    turns[i] = theta * 0.15915494309189533577;
}

// A workgroup takes one row; D / 8 lanes a head, 8 elements a lane.  The
// row's cosines and sines are taken once, by rot / 2 threads, and shared by
// its heads through LDS (a copy a head would cost 40 times the 64-bit
// reductions).  Lanes u < rot / 8 of a head hold four whole pairs -- elements
// 4 u .. and rot / 2 + 4 u .. (neox), or 8 u .. -- so a pair never crosses a
// lane; the others hold 8 elements behind the turned part.  Memory-bound: 4
// bytes in and 2 out an element, all of it in 16- and 8-byte pieces.  4000 rows of
// 48 heads of 128: 31 us, 4.7 TB/s; one row 3.0 us.
template <int D, bool NEOX>
__global__ __launch_bounds__(256) void rf_paged_rope_kernel(const rf_paged_rope s, const rf_paged_cache c) {
    constexpr int LPH = D / 8, HPB = 256 / LPH;
    __shared__ float2 cs[D / 2];
    const int r = blockIdx.x;
    const int slot = s.slots[r];
    if (slot < 0 || slot >= c.num_pages * c.page_size) return;
    const int tid = threadIdx.x, u = tid % LPH, heads = s.num_heads + 2 * c.num_kv_heads;
    const int half = s.rot_dim / 2;
    const bool turned = u < s.rot_dim / 8;
    const int e0 = NEOX && turned ? 4 * u : 8 * u, e1 = NEOX && turned ? half + 4 * u : e0 + 4;
    const int64_t at = (int64_t)(slot / c.page_size) * c.page_stride + (slot % c.page_size) * c.row_stride;

    const int first = blockIdx.y * HPB + tid / LPH, step = gridDim.y * HPB;
    float4 a, b;
    auto load = [&](int h) {
        const float* src = h < s.num_heads ? s.q + r * s.ld_q + (int64_t)h * D
                           : h < s.num_heads + c.num_kv_heads
                               ? s.k + r * s.ld_k + (int64_t)(h - s.num_heads) * D
                               : s.v + r * s.ld_v + (int64_t)(h - s.num_heads - c.num_kv_heads) * D;
        a = *reinterpret_cast<const float4*>(src + e0);
        b = *reinterpret_cast<const float4*>(src + e1);
    };
    if (first < heads) load(first);
    if (tid < half) {
        const double turn = (double)s.positions[r] * s.turns[tid];
        float sn, co;
        sincospif(2.0f * (float)(turn - rint(turn)), &sn, &co);
        cs[tid] = make_float2(co * s.attn_factor, sn * s.attn_factor);
    }
    __syncthreads();
    for (int h = first; h < heads; h += step) {
        float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        if (h + step < heads) load(h + step);
        const bool is_q = h < s.num_heads, is_v = h >= s.num_heads + c.num_kv_heads;
        const float* w = is_v ? nullptr : is_q ? s.q_norm : s.k_norm;
        // (every lane of a head takes the same way, and heads do not share lanes)
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __fmaf_rn(x[i], x[i], ss);
        ss = xor_sum<LPH / 2, 1>(ss);
        if (w != nullptr) {
            const float inv = 1.0f / sqrtf(ss * (1.0f / D) + s.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[(i < 4 ? e0 : e1 - 4) + i];
        }
        if (!is_v && turned) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 w2 = cs[4 * u + i];
                constexpr int P = NEOX ? 1 : 2, Q = NEOX ? 4 : 1;
                const float p = x[P * i], q = x[P * i + Q];
                x[P * i] = __fmaf_rn(p, w2.x, -(q * w2.y));
                x[P * i + Q] = __fmaf_rn(p, w2.y, q * w2.x);
            }
        }
        uint16_t* dst = is_q   ? s.q16 + r * s.ld_q16 + (int64_t)h * D
                        : is_v ? c.v + at + (h - s.num_heads - c.num_kv_heads) * c.head_stride
                               : c.k + at + (h - s.num_heads) * c.head_stride;
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = (uint32_t)f16_bits_rn(x[2 * i]) | ((uint32_t)f16_bits_rn(x[2 * i + 1]) << 16);
        *reinterpret_cast<uint2*>(dst + e0) = make_uint2(o[0], o[1]);
        *reinterpret_cast<uint2*>(dst + e1) = make_uint2(o[2], o[3]);
    }
}

// ---- rules on the logits -------------------------------------------------------------------
//
// A workgroup takes kSlice tokens of one row: it starts their loads, counts
// the history's tokens that fall among them in LDS (integers, so the order of
// the atomics does not matter), marks the bias list's, and writes the slice in
// one pass; a marked token's wave adds up its entries in list order.  The
// history is read once a slice, from L2.  Bound: 8 bytes a token, and for few
// rows the latency of history and logits.  64 rows of 151936 tokens, masked, 1 to
// 8000 tokens of history: 23 us, 3.5 TB/s; one row with 4000 6 us.  Up to 64 entries of the
// bias list among a slice's tokens are kept beside it; with more, every marked token's
// wave reads the row's list again, which grows with its square: 64 rows and 300 /
// 1000 / 2000 / 10,000 entries each, over the whole vocabulary, 20 / 24 / 159 / 4400 us (no list 15).
// of a token in LDS: its place in the history, a mark for the bias list, a count of those not in the prompt
constexpr uint32_t kSeen = 1, kBiased = 2, kMade = 4;

template <bool VEC, int kSlice>
__global__ __launch_bounds__(256) void rf_logits_rules_kernel(const rf_logits_rules l) {
    __shared__ __align__(16) uint32_t count[kSlice];        // (cleared in 16 bytes)
    __shared__ int listed, list_at[64], list_id[64];
    __shared__ float list_val[64];
    constexpr int IDS = 8;                       // of the history in flight a thread
    constexpr int V = VEC ? 4 : 1, N = kSlice / (256 * V);
    const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, base = blockIdx.x * kSlice;
    const int n = min(kSlice, l.vocab - base);   // tokens of this slice
    const float* x = l.logits + r * l.ld_logits + base;
    float* y = l.out + r * l.ld_out + base;
    // (plain loads and no restrict: out may be logits, each element read and written by its own thread)
    float v[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = (i * 256 + tid) * V;
        if (VEC && e + 3 < n) {
            const float4 q = *reinterpret_cast<const float4*>(x + e);
            v[i][0] = q.x;
            v[i][V > 1 ? 1 : 0] = V > 1 ? q.y : q.x;
            v[i][V > 2 ? 2 : 0] = V > 2 ? q.z : q.x;
            v[i][V > 3 ? 3 : 0] = V > 3 ? q.w : q.x;
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) v[i][k] = e + k < n ? x[e + k] : 0.0f;
        }
    }
    const bool penal = l.repetition != nullptr || l.frequency != nullptr || l.presence != nullptr;
    const int64_t total = penal ? min((int64_t)max(l.total_lens[r], 0), l.ld_history) : 0;
    const int prompt = penal ? l.prompt_lens[r] : 0;
    const int b0 = l.bias_start != nullptr ? max(l.bias_start[r], 0) : 0;
    const int b1 = l.bias_start != nullptr ? l.bias_start[r + 1] : 0;
    for (int i = tid; i < kSlice / 4; i += 256) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) listed = 0;
    __syncthreads();
    const int* hist = l.history + r * l.ld_history;
    for (int64_t i0 = tid; i0 < total; i0 += 256 * IDS) {
        uint32_t id[IDS];
#pragma unroll
        for (int k = 0; k < IDS; ++k) id[k] = i0 + 256 * k < total ? (uint32_t)hist[i0 + 256 * k] - (uint32_t)base : ~0u;
#pragma unroll
        for (int k = 0; k < IDS; ++k)
            if (id[k] < (uint32_t)n) {
                if (i0 + 256 * k >= prompt)
                    atomicAdd(&count[id[k]], kMade);
                else
                    atomicOr(&count[id[k]], kSeen);
            }
    }
    for (int j = b0 + tid; j < b1; j += 256) {
        const uint32_t id = (uint32_t)l.bias_ids[j] - (uint32_t)base;
        if (id < (uint32_t)n) {
            atomicOr(&count[id], kBiased);
            const int k = atomicAdd(&listed, 1);
            if (k < 64) {
                list_at[k] = j;
                list_id[k] = (int)id;
                list_val[k] = l.bias_values[j];
            }
        }
    }
    __syncthreads();
    // the slice's entries of the bias list, one a lane, in any order
    const bool short_list = listed <= 64;
    const bool mine = short_list && lane < listed;
    const int my_at = mine ? list_at[lane] : INT_MAX, my_id = mine ? list_id[lane] : -1;
    const float my_val = mine ? list_val[lane] : 0.0f;
    const float rep = l.repetition != nullptr ? l.repetition[r] : 1.0f;
    const float freq = l.frequency != nullptr ? l.frequency[r] : 0.0f;
    const float pres = l.presence != nullptr ? l.presence[r] : 0.0f;
    const uint32_t* allowed = l.allowed != nullptr ? l.allowed + r * l.ld_allowed + base / 32 : nullptr;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = (i * 256 + tid) * V;
        uint32_t c[V];
#pragma unroll
        for (int k = 0; k < V; ++k) c[k] = count[e + k];
        const uint32_t bits = allowed != nullptr && e < n ? allowed[e / 32] >> (e % 32) : ~0u;
        float o[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float z = v[i][k];
            if (c[k] & ~kBiased) {
                if (l.repetition != nullptr) z = z > 0.0f ? z / rep : z * rep;
                if (c[k] >= kMade) z = (z - freq * (float)(c[k] / kMade)) - pres;
            }
            o[k] = z;
        }
        if (listed > 0) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                uint64_t marked = __ballot(c[k] & kBiased);
                while (marked) {                 // token by token, its entries in list order
                    const int to = __builtin_ctzll(marked);
                    marked &= marked - 1;
                    const int id = __shfl(e, to) + k;
                    float sum = 0.0f;
                    if (short_list) {
                        uint64_t hits = __ballot(my_id == id);
                        while (hits) {
                            int next = __builtin_ctzll(hits);
                            for (uint64_t rest = hits & (hits - 1); rest; rest &= rest - 1)
                                if (__shfl(my_at, __builtin_ctzll(rest)) < __shfl(my_at, next))
                                    next = __builtin_ctzll(rest);
                            sum += __shfl(my_val, next);
                            hits &= ~(1ull << next);
                        }
                    } else {
                        for (int j0 = b0; j0 < b1; j0 += 64) {
                            const bool there = j0 + lane < b1;
                            const bool same = there && l.bias_ids[there ? j0 + lane : b0] == base + id;
                            uint64_t hits = __ballot(same);
                            const float val = same ? l.bias_values[j0 + lane] : 0.0f;
                            for (; hits; hits &= hits - 1) sum += __shfl(val, __builtin_ctzll(hits));
                        }
                    }
                    if (lane == to) o[k] += sum;
                }
            }
        }
        if (e >= n) continue;
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = (bits >> k) & 1u ? o[k] : -INFINITY;
        if (VEC && e + 3 < n) {
            *reinterpret_cast<float4*>(y + e) = make_float4(o[0], o[V > 1 ? 1 : 0], o[V > 2 ? 2 : 0], o[V > 3 ? 3 : 0]);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (e + k < n) y[e + k] = o[k];
        }
    }
}

}  // namespace rf

// ---- launchers -----------------------------------------------------------------------------

static bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Up to kPlanRows rows the scanning workgroup writes them itself.
static constexpr int kPlanRows = 8192;

extern "C" hipError_t rf_paged_plan_launch(const rf_paged_plan* plan, hipStream_t stream) {
    if (plan == nullptr) return hipErrorInvalidValue;
    const rf_paged_plan& p = *plan;
    if (p.num_seqs < 0 || p.max_rows < 0 || p.max_blocks < 0 || p.num_pages < 0 || !rf::page_size_ok(p.page_size) ||
        (int64_t)p.num_pages * p.page_size > INT_MAX)
        return hipErrorInvalidValue;
    if (p.num_seqs == 0 && p.max_rows == 0) return hipSuccess;
    if (!p.q_start || !p.free_in || !p.free_out || (p.max_rows > 0 && (!p.positions || !p.slots)) ||
        (p.num_seqs > 0 && (!p.new_lens || !p.ctx_in || !p.ctx_out || !p.kv_lens || !p.block_tables || !p.free_pages)))
        return hipErrorInvalidValue;
    if (p.max_rows <= kPlanRows && p.num_seqs <= rf::kPlanThreads) {
        hipLaunchKernelGGL(rf::rf_paged_plan_kernel<true>, dim3(1), dim3(rf::kPlanThreads), 0, stream, p);
    } else {
        hipLaunchKernelGGL(rf::rf_paged_plan_kernel<false>, dim3(1), dim3(rf::kPlanThreads), 0, stream, p);
        if (p.max_rows > 0)
            hipLaunchKernelGGL(rf::rf_paged_rows_kernel, dim3((unsigned)(((int64_t)p.max_rows + 255) / 256)), dim3(256),
                               0, stream, p);
    }
    return hipGetLastError();
}

extern "C" hipError_t rf_paged_release_launch(const int32_t* ended, int32_t* ctx_lens, const int32_t* block_tables,
                                              int32_t* free_pages, int32_t* free_count, int num_seqs, int max_blocks,
                                              int page_size, int num_pages, hipStream_t stream) {
    if (num_seqs < 0 || max_blocks < 0 || num_pages < 0 || !rf::page_size_ok(page_size)) return hipErrorInvalidValue;
    if (num_seqs == 0) return hipSuccess;
    if (!ended || !ctx_lens || !block_tables || !free_pages || !free_count) return hipErrorInvalidValue;
    hipLaunchKernelGGL(rf::rf_paged_release_kernel, dim3(1), dim3(rf::kPlanThreads), 0, stream, ended, ctx_lens,
                       block_tables, free_pages, free_count, num_seqs, max_blocks, page_size, num_pages);
    return hipGetLastError();
}

extern "C" hipError_t rf_rope_turns_table(double* d_turns, int rot_dim, double theta_base, int mode, double factor,
                                          double orig_positions, double beta_fast, double beta_slow,
                                          const float* d_freq_scale, hipStream_t stream) {
    if (!d_turns || rot_dim < 2 || rot_dim > 256 || rot_dim % 2 || !(theta_base > 1.0) || !(factor > 0.0) ||
        !std::isfinite(theta_base) || !std::isfinite(factor) || mode < RF_ROPE_PLAIN || mode > RF_ROPE_YARN)
        return hipErrorInvalidValue;
    double lo = 0.0, hi = 0.0;
    if (mode == RF_ROPE_YARN) {
        if (!(orig_positions > 0.0) || !(beta_slow > 0.0) || !(beta_fast >= beta_slow) || !std::isfinite(beta_fast) ||
            !std::isfinite(orig_positions))
            return hipErrorInvalidValue;
        const double two_pi = 6.283185307179586477;
        lo = std::fmax(std::floor(rot_dim * std::log(orig_positions / (beta_fast * two_pi)) / (2.0 * std::log(theta_base))),
                       0.0);
        hi = std::fmin(std::ceil(rot_dim * std::log(orig_positions / (beta_slow * two_pi)) / (2.0 * std::log(theta_base))),
                       rot_dim - 1.0);
    }
    hipLaunchKernelGGL(rf::rf_rope_turns_kernel, dim3(1), dim3(128), 0, stream, d_turns, rot_dim, theta_base, mode,
                       factor, lo, hi, d_freq_scale);
    return hipGetLastError();
}

extern "C" hipError_t rf_paged_rope_write_launch(const rf_paged_rope* step, const rf_paged_cache* cache,
                                                 hipStream_t stream) {
    if (step == nullptr || cache == nullptr) return hipErrorInvalidValue;
    const rf_paged_rope& s = *step;
    if (!rf::cache_ok(*cache) || s.rows < 0 || s.rows > (1 << 23) || s.num_heads <= 0 || s.num_heads > 65535 ||
        s.rot_dim < 0 || s.rot_dim > cache->head_dim || s.rot_dim % 8)
        return hipErrorInvalidValue;
    if (s.rows == 0) return hipSuccess;
    if (!s.q || !s.k || !s.v || !s.q16 || !s.positions || !s.slots || (s.rot_dim > 0 && !s.turns))
        return hipErrorInvalidValue;
    if (!aligned(s.q, 16) || !aligned(s.k, 16) || !aligned(s.v, 16) || !aligned(s.q16, 16) || !aligned(s.q_norm, 16) ||
        !aligned(s.k_norm, 16) || !aligned(s.turns, 8) || s.ld_q % 4 || s.ld_k % 4 || s.ld_v % 4 || s.ld_q16 % 8 ||
        s.ld_q < 0 || s.ld_k < 0 || s.ld_v < 0 || s.ld_q16 < (int64_t)s.num_heads * cache->head_dim)
        return hipErrorInvalidValue;
    const int heads = s.num_heads + 2 * cache->num_kv_heads, hpb = 256 / (cache->head_dim / 8);
    const int passes = (heads + hpb - 1) / hpb;
    // few rows: a row's heads over several workgroups, each with the row's cosines
    const int split = s.rows * (int64_t)passes <= 2 * rf::device_cu_count() ? passes : 1;
    const dim3 grid(s.rows, split), blk(256);
#define ROPE_GO(D)                                                                                    \
    if (s.neox)                                                                                       \
        hipLaunchKernelGGL((rf::rf_paged_rope_kernel<D, true>), grid, blk, 0, stream, s, *cache);     \
    else                                                                                              \
        hipLaunchKernelGGL((rf::rf_paged_rope_kernel<D, false>), grid, blk, 0, stream, s, *cache);
    switch (cache->head_dim) {
    case 64: ROPE_GO(64) break;
    case 128: ROPE_GO(128) break;
    default: ROPE_GO(256) break;
    }
#undef ROPE_GO
    return hipGetLastError();
}

extern "C" hipError_t rf_logits_rules_launch(const rf_logits_rules* rules, hipStream_t stream) {
    if (rules == nullptr) return hipErrorInvalidValue;
    const rf_logits_rules& l = *rules;
    if (l.rows < 0 || l.rows > 65535 || l.vocab < 0) return hipErrorInvalidValue;
    if (l.rows == 0 || l.vocab == 0) return hipSuccess;
    const bool penal = l.repetition || l.frequency || l.presence;
    const int bias = !!l.bias_start + !!l.bias_ids + !!l.bias_values;
    if (!l.logits || !l.out || l.ld_logits < l.vocab || l.ld_out < l.vocab || (bias != 0 && bias != 3) ||
        (penal && (!l.history || !l.prompt_lens || !l.total_lens || l.ld_history < 0)) ||
        (l.allowed && l.ld_allowed < (l.vocab + (int64_t)31) / 32) || (l.out == l.logits && l.ld_out != l.ld_logits))
        return hipErrorInvalidValue;
    const bool vec = l.ld_logits % 4 == 0 && l.ld_out % 4 == 0 && aligned(l.logits, 16) && aligned(l.out, 16);
    // slices of 4096 tokens (the history is read once each), of 1024 where those leave CUs idle
    const auto slices = [&](int n) { return (unsigned)((l.vocab + (int64_t)n - 1) / n); };
    const bool few = (int64_t)l.rows * slices(4096) < rf::device_cu_count();
    const dim3 grid(slices(few ? 1024 : 4096), l.rows), blk(256);
    if (vec && few)
        hipLaunchKernelGGL((rf::rf_logits_rules_kernel<true, 1024>), grid, blk, 0, stream, l);
    else if (vec)
        hipLaunchKernelGGL((rf::rf_logits_rules_kernel<true, 4096>), grid, blk, 0, stream, l);
    else if (few)
        hipLaunchKernelGGL((rf::rf_logits_rules_kernel<false, 1024>), grid, blk, 0, stream, l);
    else
        hipLaunchKernelGGL((rf::rf_logits_rules_kernel<false, 4096>), grid, blk, 0, stream, l);
    return hipGetLastError();
}
