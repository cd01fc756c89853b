// paged8_attn.hip -- causal GQA attention of the new rows of a batch over 8-bit
// pages (rf_paged_attention8_launch; the header states what it computes,
// paged_attn.h how a batch is cut).  No counterpart in the reference.
//
// Codes become fp16 values, exactly, on their way into the MFMAs: both the fp16
// kernels' sums and their rules for masks, infinities and NaN hold as they are.
#include "paged8.h"
#include "paged_attn.h"

namespace rf {

typedef int i2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i2* lds_i2;
typedef __attribute__((address_space(3))) const u32x4* lds_u4;
typedef __attribute__((address_space(3))) float* lds_f;
typedef __attribute__((address_space(3))) const int* lds_int;

// A row of D codes in LDS lies as in memory, its 16-byte pieces permuted so that neither
// K's reads (one piece of 16 rows) nor V's transposing ones (one piece of the rows 8 i .. 8 i + 7
// and 16 further, i = 0 or 1) meet a bank twice; 256 / D rows fill the banks.
template <int D>
__device__ __forceinline__ int k_swizzle8(int row) {
    return D == 64 ? (row >> 2) & 3 : D == 128 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_swizzle8(int row) {
    const int far = (row >> 4) & 1;
    return D == 64 ? ((row >> 2) & 1) | (far << 1) : D == 128 ? ((row >> 1) & 3) | (far << 2) : (row & 7) | (far << 3);
}

// 16 bytes a lane from each lane's own address into LDS at m0 + 16 lane
__device__ __forceinline__ void lds_dma16_at(uint32_t lds_dst, uint64_t at) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_dst), "v"(at) : "memory", "m0");
}

// A byte a lane, as 32 bits at m0 + 4 lane
__device__ __forceinline__ void lds_dma_byte_at(uint32_t lds_dst, uint64_t at) {
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_ubyte %1, off" ::"s"(lds_dst), "v"(at) : "memory", "m0");
}

// ---- few rows -------------------------------------------------------------------------
//
// find_share's items in another order, for 17 to 64 requests: those of the longest parts first, in eighths of
// a share, so that short ones fill the end of a launch.  48 requests of 60 to 16000 positions 49.2 us, in the
// requests' order 52.6, 32 of 100 to 8000 24.5 and 27.3; for few requests it is 0.2 us of instructions.
template <int ROWS, int KEYS>
__device__ __forceinline__ bool find_longest(const rf_paged_attention& a, const rf_paged_cache8& c, const Plan& p, int j,
                                             Share& s) {
    const Request r = request_of<ROWS, KEYS>(a, c, p, threadIdx.x & 63);
    const int share = share_of<ROWS, KEYS>(a, c, p, r);
    const int parts = max((int)(((unsigned)r.units + share - 1) / (unsigned)share), 1), items = r.tiles * parts;
    const int slots = parts > 1 ? items : 0, slots_end = wave_scan(slots);
    const int length = (int)min(8ll * r.units / ((int64_t)parts * share), 7ll);
    for (int k = 7; k >= 0; --k) {
        const int mine = length == k ? items : 0, end = wave_scan(mine), all = __builtin_amdgcn_readlane(end, 63);
        if (j >= all) {
            j -= all;
            continue;
        }
        const int l = __builtin_ctzll(__ballot(end > j));
        auto get = [l](int v) { return __builtin_amdgcn_readlane(v, l); };
        s.b = l;
        s.q0 = get(r.q0);
        s.n = get(r.n);
        s.kv = get(r.kv);
        s.tiles = get(r.tiles);
        s.parts = get(parts);
        s.slot = get(slots_end - slots);
        const int at = j - get(end - mine);
        s.part = at / s.tiles;
        s.tile = s.tiles - 1 - (at - s.part * s.tiles);
        return true;
    }
    return false;
}

// As over fp16 pages (paged_attn.hip): wave w takes the pieces of 32 positions w, w + W, .. of
// the part through its own S-stage ring in LDS, codes as they are; they become fp16 in
// registers, K's under its row's exponent and V's under their keys' (lane 4 i + j of a window
// of 16 pieces holds address and exponents of piece i's unit j of 8 positions).
template <int D, int W, int S>
__device__ __forceinline__ void narrow8_part(const rf_paged_attention& a, const rf_paged_cache8& c, const Plan& plan,
                                             int item, uint8_t* lds) {
    constexpr int MAT = kNarrowKeys * D, STAGE = 2 * MAT;
    constexpr int LPR = D / 16, RPI = 64 / LPR, NI = kNarrowKeys / RPI;           // lanes a row, rows an instruction
    constexpr int KS = D / 32, NB = D / 16;
    constexpr int PADD = D + 4;                          // floats a row of the join
    static_assert(kNarrowRows * (PADD + 2) * 4 <= S * STAGE, "the join fits the ring");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int nkv = c.num_kv_heads;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const uint32_t ring = lds0 + (uint32_t)wave * (S * STAGE);
    const int dr = lane / LPR, ds = lane % LPR;

    Share s;
    const int kvh = item % nkv;
    if (!(a.num_seqs > 16 && a.num_seqs <= 64 ? find_longest<kNarrowRows, kNarrowKeys>(a, c, plan, item / nkv, s)
                           : find_share<kNarrowRows, kNarrowKeys>(a, c, plan, item / nkv, false, s)))
        return;
    const int rows = s.n * plan.group, r0 = kNarrowRows * s.tile;
    const Span t = span_of(plan, s, r0, min(r0 + kNarrowRows, rows) - 1, a.window);
    // the part's pieces
    const int p0 = t.lo / kNarrowKeys, p1 = (t.hi + kNarrowKeys - 1) / kNarrowKeys;
    const int each = (max(p1 - p0, 0) + s.parts - 1) / s.parts;
    const int begin = p0 + s.part * each, end = min(begin + each, p1);
    const int steps = max((end - begin - wave + W - 1) / W, 0);
    // this lane's packed row
    const int r = r0 + col, token = token_of(plan, min(r, rows - 1)), head = min(r, rows - 1) - token * plan.group;
    const int pos = s.kv - s.n + token;
    const Units<rf_paged_cache8> units(a, c, s.b, kvh, t.lo, t.hi);
    const int bsh = block_shift(c);
    bool bad = false;
    int window = 0;
    uint64_t address = 0;
    int scales = 0, scales_before = 0;                   // K's and V's byte; of the window before, whose pieces may still wait
    const uint64_t v_from_k = (uint64_t)c.v - (uint64_t)c.k;
    const uint32_t stride = (uint32_t)c.row_stride;
    auto load_units = [&](int step) {
        const int unit = 4 * (begin + wave + W * (step + (lane >> 2))) + (lane & 3);
        const int page = units.page_of(unit);
        address = units.address(unit, page, bad);
        const int64_t at = scale_at(c, (unsigned)page >= (unsigned)c.num_pages ? 0 : page,
                                    (8 * units.seen(unit)) & units.pmask, bsh) + kvh;
        scales_before = scales;
        scales = scale_byte(c.k_scale[at]) | (scale_byte(c.v_scale[at]) << 8);
        window = step;
    };
    auto stage = [&](int step) {
        if (step >= steps) return;
        if (step - window >= 16) load_units(step);
        const int piece = begin + wave + W * step, k0 = kNarrowKeys * piece;
        const uint32_t dst = ring + (uint32_t)(step % S) * STAGE;
        const bool whole = k0 >= t.lo && k0 + kNarrowKeys <= t.hi;
        // the ring's last readers are done
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int lr = RPI * i + dr;
            const uint32_t kp = 16u * (uint32_t)(ds ^ k_swizzle8<D>(lr)), vp = 16u * (uint32_t)(ds ^ v_swizzle8<D>(lr));
            const uint32_t kd = __builtin_amdgcn_readfirstlane(dst + 1024u * i);
            const uint32_t vd = __builtin_amdgcn_readfirstlane(dst + MAT + 1024u * i);
            // positions that no row sees are taken from the nearest one that some row sees
            if constexpr (RPI > 8) {
                // two units an instruction
                const int key = whole ? k0 + lr : min(max(k0 + lr, t.lo), t.hi - 1);
                const uint64_t lo = read_lane(address, 4 * (step - window) + 2 * i);
                const uint64_t hi = read_lane(address, 4 * (step - window) + 2 * i + 1);
                const int unit = units.seen(4 * piece + 2 * i + (lane >> 5));
                const uint64_t at = (lane < 32 ? lo : hi) + (uint64_t)((uint32_t)(key - 8 * unit) * stride);
                lds_dma16_at(kd, at + kp);
                lds_dma16_at(vd, at + v_from_k + vp);
            } else {
                int unit = 4 * piece + (RPI * i >> 3);
                uint32_t row = (uint32_t)((RPI * i & 7) + dr) * stride;
                if (!whole) {
                    unit = units.seen(unit);
                    row = (uint32_t)(min(max(k0 + lr, t.lo), t.hi - 1) - 8 * unit) * stride;
                }
                const uint64_t at = read_lane(address, 4 * (step - window) + unit - 4 * piece);
                lds_dma16(kd, row + kp, reinterpret_cast<const uint8_t*>(at));
                lds_dma16(vd, row + vp, reinterpret_cast<const uint8_t*>(at + v_from_k));
            }
        }
    };
    // dims 64 j + 16 quad + {0 .. 7, 8 .. 15} are this lane's of k-steps 2 j and 2 j + 1, as K's 16-byte reads have them
    h8 q[KS];
    const uint16_t* qrow = a.q + (int64_t)(s.q0 + token) * a.ld_q + (int64_t)(kvh * plan.group + head) * D + 16 * quad;
#pragma unroll
    for (int k = 0; k < KS; ++k) q[k] = *reinterpret_cast<const h8*>(qrow + 64 * (k >> 1) + 8 * (k & 1));
    if (steps > 0) load_units(0);
    // (q has arrived before the DMAs start, so that none but theirs are counted below)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < S - 1; ++i) stage(i);

    // operand addresses: one base and an xor each
    const uint32_t ka = ring + (uint32_t)col * D + 16u * (uint32_t)(quad ^ k_swizzle8<D>(col));
    const int vr = 4 * quad + ((col >> 1) & 3) + 16 * (col >> 3);
    const uint32_t va = ring + MAT + (uint32_t)vr * D + 16u * (uint32_t)v_swizzle8<D>(vr) + 8u * (uint32_t)(col & 1);

    const float scale = a.scale * kLog2e;
    f4 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f4{0, 0, 0, 0};
    float m = kNone, l = 0.0f;
    bool dirty = false;
    for (int step = 0; step < steps; ++step) {
        stage(step + S - 1);
        if (step + S <= steps)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * 2 * NI) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const int k0 = kNarrowKeys * (begin + wave + W * step);
        const uint32_t at = (uint32_t)(step % S) * STAGE;
        // (opaque, so that a piece's addresses are not kept in registers over the loop)
        uint32_t kt = ka + at, vt = va + at;
        asm("" : "+v"(kt), "+v"(vt));
        // the exponents: K's of rows col and 16 + col, V's of keys 4 quad .. and 16 + 4 quad ..
        const int held = step >= window ? scales : scales_before, w0 = 4 * (step & 15);
        auto of_unit = [&](int unit) { return __builtin_amdgcn_ds_bpermute(4 * (w0 + unit), held); };
        float ks[2], vs[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            ks[b] = pow2_of(of_unit(2 * b + (col >> 3)) & 0xff);
            vs[b] = pow2_of(of_unit(2 * b + (quad >> 1)) >> 8);
        }
        f4 x[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int j = 0; j < KS / 2; ++j)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                h8 lo, hi;
                values_of(*(lds_u4)((kt ^ (64u * j)) + 16u * b * D), ks[b], lo, hi);
                x[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, q[2 * j], x[b], 0, 0, 0);
                x[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, q[2 * j + 1], x[b], 0, 0, 0);
            }
        const bool masked = k0 + kNarrowKeys - 1 > t.first || (a.window > 0 && k0 <= t.last - a.window);
        const int ahead = pos - k0 - 4 * quad, behind = a.window > 0 ? ahead - a.window : INT_MIN;
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[b][e] *= scale;
                if (masked && (16 * b + e > ahead || 16 * b + e <= behind)) x[b][e] = -INFINITY;
                top = fmaxf(top, x[b][e]);
            }
        top = xor_butterfly<32, 16>(top, max_raw);
        const bool up = top > m + (kLag + kLift);
        if (__ballot(up)) {
            const float f = up ? __builtin_amdgcn_exp2f(m - (top - kLift)) : 1.0f;
            m = up ? top - kLift : m;
            l *= f;
#pragma unroll
            for (int i = 0; i < NB; ++i) o[i] *= f;
        }
        h8 p;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) p[4 * b + e] = (_Float16)__builtin_amdgcn_exp2f(x[b][e] - m);
        l += sum8(p, 0.0f);
        // V^T: lane (dim 16 i + col) takes keys 4 quad + {0 .. 3, 16 .. 19}, as p holds them.  NaN
        // among values that some rows do not see must not meet their zero weights: finite values
        // take its place, and the rows that see it get it at the end.
        Finite fin;
#pragma unroll
        for (int i0 = 0; i0 < NB; i0 += 4) {
            h8 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const i2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2)(vt ^ (16u * (i0 + i))));
                v[i] = join(__builtin_shufflevector(two_of<false>(w[0], vs[0]), two_of<true>(w[0], vs[0]), 0, 1, 2, 3),
                            __builtin_shufflevector(two_of<false>(w[1], vs[1]), two_of<true>(w[1], vs[1]), 0, 1, 2, 3));
            }
            if (masked) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    fin.take(v[i]);
                    v[i] = finite_of(v[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[i0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[i], p, o[i0 + i], 0, 0, 0);
        }
        if (masked) dirty = dirty || !fin.all();
    }
    if (dirty) {
        // the NaN that were replaced, to the rows that see them
        const uint8_t* vc = c.v + kvh * c.head_stride;
#pragma unroll 1
        for (int k0 = kNarrowKeys * begin; k0 < kNarrowKeys * end; ++k0) {
            const int k32 = k0 & ~31;
            if (k32 / kNarrowKeys % W != (begin + wave) % W || k0 < t.lo || k0 >= t.hi) continue;
            if (!(k32 + 31 > t.first || (a.window > 0 && k32 <= t.last - a.window))) continue;
            const int page = units.table[k0 >> units.psh];
            if ((unsigned)page >= (unsigned)c.num_pages) continue;
            const uint8_t* row = vc + (int64_t)page * c.page_stride + (int64_t)(k0 & units.pmask) * c.row_stride + 4 * quad;
            const bool seen = k0 <= pos && (a.window == 0 || k0 > pos - a.window);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(row + 16 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] = seen && ((w >> (8 * e)) & 0x7f) == 0x7f ? NAN : o[i][e];
            }
        }
    }
    l = xor_sum<32, 16>(l);
    if (bad) l = NAN;
    // the waves' states
    float* join_o = reinterpret_cast<float*>(lds);
    float* join_m = join_o + W * kNarrowRows * PADD;
    float* join_l = join_m + W * kNarrowRows;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NB; ++i)
        *reinterpret_cast<f4*>(join_o + (wave * kNarrowRows + col) * PADD + 16 * i + 4 * quad) = o[i];
    if (quad == 0) {
        join_m[wave * kNarrowRows + col] = m;
        join_l[wave * kNarrowRows + col] = l;
    }
    __syncthreads();
    const int live = min(rows - r0, kNarrowRows);
    float* part = slot_of<kNarrowRows, D>(plan.states, s, s.part, kvh, nkv);
    for (int i = threadIdx.x; i < live * (D / 4); i += 64 * W) {
        const int row = i / (D / 4), d = 4 * (i % (D / 4));
        float mx = kNone, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) mx = fmaxf(mx, join_m[w * kNarrowRows + row]);
        f4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = __builtin_amdgcn_exp2f(join_m[w * kNarrowRows + row] - mx);
            sum += join_l[w * kNarrowRows + row] * f;
            acc += *reinterpret_cast<f4*>(join_o + (w * kNarrowRows + row) * PADD + d) * f;
        }
        if (s.parts > 1) {
            *reinterpret_cast<f4*>(part + row * D + d) = acc;
            if (d == 0) {
                part[kNarrowRows * D + row] = mx;
                part[kNarrowRows * (D + 1) + row] = sum;
            }
        } else {
            const int tk = token_of(plan, r0 + row), hd = r0 + row - tk * plan.group;
            // (a row in front of position 0 sees nothing; one whose scores are all -inf is 0 / 0)
            store4(a, (int64_t)(s.q0 + tk) * a.ld_out + (int64_t)(kvh * plan.group + hd) * D + d,
                   s.kv - s.n + tk < 0 ? f4{0, 0, 0, 0} : acc * (1.0f / sum));
        }
    }
}

// ---- pieces of prompt, heads of 256 ---------------------------------------------------------
//
// Two waves share 32 packed rows: each has the scores of half of a tile's 64 positions and the
// outputs of half of the dims, and they swap weights through LDS, in the registers' order.  So a
// wave's queries and outputs take 128 registers, two waves fit a SIMD, and an operand that is
// read from LDS meets 32 rows.  Codes stay codes in LDS and become fp16 on their way into the MFMAs:
// an operand's conversion is 16 clocks of VALU beside the 32 of its MFMA.  Three stages of tiles: with two,
// each turn waited for memory.  A turn of 64 positions takes 2.16 us, some 5000 clocks, where its MFMAs take 2048 and
// its VALU instructions 2700 a SIMD, in two waves that overlap little; a step of three windowed prompts
// 70 us, with 16 rows a wave over fp16 values in LDS 106; 512 tokens behind 62800 positions 564 us, 940 TFLOP/s.
//
// A row's maximum is rounded up to a whole number, so that the two waves' weights come to the
// larger one by powers of two, exactly but for those that become subnormal.  No weight of a row need be one of
// fp16's then, so the sum is of the weights before they are rounded: an output is off by their roundings, 2^-11
// of sum w |v| at most, where a sum of rounded weights would let two comparable ones err by twice that.  A row of
// one key has its value all the same: its sum, that one weight, is rounded at the end.
constexpr int kPairRows = 32, kPairStages = 3;
template <int D, int NW>
constexpr int pair8_lds() { return 2 * kPairStages * kWideKeys * D + NW * (2 * 2048 + 3 * 4 * kPairRows) + 1024; }

// Dims of 4 part + {0 .. 3, 8 .. 11} positions of 16: rows of 16 bytes, the 16 lanes' 8 rows and the
// next piece's in other banks.
__device__ __forceinline__ uint32_t pair_swizzle(uint32_t row) { return 2 * ((row & 3) | ((row >> 1) & 4)); }

// find_share's items in another order, for up to 64 requests: those that a window makes equally long in the
// requests' order, then the first (longest) of the others of each request, the second of each, and
// so on, so that short ones fill the end of a launch.  16 heads on 8, window 1024: three prompts of 600 to
// 1900 tokens and six single ones 72 us, in the requests' order 80; four of 100 to 3000 69 and 71 (all of
// them by rank 15 more: neighbours share K and V in an XCD's L2); eight of 200 to 1000 behind up to 6000 positions
// without a window 135 and 144, but eight fresh ones 64.5 and 61.
template <int ROWS, int KEYS>
__device__ __forceinline__ bool find_ranked(const rf_paged_attention& a, const rf_paged_cache8& c, const Plan& p, int j,
                                            Share& s) {
    const Request r = request_of<ROWS, KEYS>(a, c, p, threadIdx.x & 63);
    const int share = share_of<ROWS, KEYS>(a, c, p, r);
    const int parts = max((int)(((unsigned)r.units + share - 1) / (unsigned)share), 1), items = r.tiles * parts;
    const int slots = parts > 1 ? items : 0, slots_end = wave_scan(slots);
    // (tiles whose rows all see from position 0 on are the shorter, the earlier they are)
    const int growing = a.window == 0 ? items : parts > 1 ? 0 : (int)max(min((int64_t)a.window - (r.kv - r.n), (int64_t)r.n), (int64_t)0) * p.group / ROWS;
    const int equal = items - growing, equal_end = wave_scan(equal), equals = __builtin_amdgcn_readlane(equal_end, 63);
    int l, at;
    if (j < equals) {
        l = __builtin_ctzll(__ballot(equal_end > j));
        at = j - __builtin_amdgcn_readlane(equal_end - equal, l);
    } else {
        j -= equals;
        const int all = wave_total(growing);
        if (j >= all) return false;
        // the rank: the last one with no more items before it, the sum of min(growing, rank)
        int lo = 0, before = 0;
        if ((__popcll(__ballot(growing > 0))) == 1) lo = before = j;
        for (int hi = all; lo < j && hi - lo > 1;) {
            const int k = (lo + hi) >> 1, n = wave_total(min(growing, k));
            if (n <= j) {
                lo = k;
                before = n;
            } else {
                hi = k;
            }
        }
        const uint64_t there = __ballot(growing > lo);
        const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(there >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)there, 0));
        l = __builtin_ctzll(__ballot(growing > lo && rank == j - before));
        at = __builtin_amdgcn_readlane(equal, l) + lo;
    }
    auto get = [l](int v) { return __builtin_amdgcn_readlane(v, l); };
    s.b = l;
    s.q0 = get(r.q0);
    s.n = get(r.n);
    s.kv = get(r.kv);
    s.tiles = get(r.tiles);
    s.parts = get(parts);
    s.slot = get(slots_end - slots);
    s.part = at / s.tiles;
    s.tile = s.tiles - 1 - (at - s.part * s.tiles);
    return true;
}

template <int D, int NW>
__device__ __forceinline__ void pair8_part(const rf_paged_attention& a, const rf_paged_cache8& c, const Plan& plan,
                                           int item, uint8_t* lds) {
    static_assert(D == 256, "a row of 16 pieces, its half a wave's outputs");
    constexpr int M = kPairRows, ROWS = M * NW / 2, MAT = kWideKeys * D, KS = D / 16, NB = D / 2 / M;
    constexpr int RPI = 4, NI = kWideKeys / (RPI * NW);          // rows an instruction, a wave's instructions a tile
    typedef Geo<M> G;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = wave & 1, col = lane % M, part = lane / M;
    // (what a lane works out from this, it works out where it is used: registers are scarce in the loop,
    // and a reload of one waits for the tiles that are on their way)
    auto lane_here = [&] {
        uint32_t l = (uint32_t)lane;
        asm volatile("" : "+v"(l));
        return l;
    };
    const int nkv = c.num_kv_heads;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const uint32_t weights0 = lds0 + 2 * kPairStages * MAT, tops0 = weights0 + 2 * NW * 2048, sums0 = tops0 + 2 * NW * 4 * M;
    const uint32_t bytes0 = sums0 + NW * 4 * M;

    Share s;
    const int kvh = item % nkv;
    if (!(a.num_seqs <= 64 ? find_ranked<ROWS, kWideKeys>(a, c, plan, item / nkv, s)
                           : find_share<ROWS, kWideKeys>(a, c, plan, item / nkv, false, s)))
        return;
    const int rows = s.n * plan.group, r0 = ROWS * s.tile;
    const Span t = span_of(plan, s, r0, min(r0 + ROWS, rows) - 1, a.window);
    const int w0 = r0 + M * (wave >> 1);
    const bool active = w0 < rows;
    const Span u = span_of(plan, s, min(w0, rows - 1), min(w0 + M, rows) - 1, a.window);
    const int p0 = t.lo / kWideKeys, p1 = (t.hi + kWideKeys - 1) / kWideKeys;
    const int each = (max(p1 - p0, 0) + s.parts - 1) / s.parts;
    const int begin = p0 + s.part * each, end = min(begin + each, p1);
    const int r = min(w0 + col, rows - 1), token = token_of(plan, r), head = r - token * plan.group;
    const int pos = s.kv - s.n + token;
    // the addresses of 64 units and the pages of the next 64; their exponents go to LDS, K's 64 and V's, with
    // the tiles (a load into a register would be waited for at the branch's end, and all tiles with it)
    const Units<rf_paged_cache8> units(a, c, s.b, kvh, t.lo, t.hi);
    const int bsh = block_shift(c);
    bool bad = false;
    int next = 0, window = -1;
    uint64_t address = 0;
    const uint64_t v_from_k = (uint64_t)c.v - (uint64_t)c.k;
    const uint32_t stride = (uint32_t)c.row_stride;
    auto bytes_at = [&](int tile) { return bytes0 + (uint32_t)(tile & 8) * 64; };
    // the buffer of the tile after one's, and of the one before
    auto after = [](uint32_t buf) { return buf == (kPairStages - 1) * MAT ? 0 : buf + MAT; };
    auto ahead_of = [](uint32_t buf) { return buf == 0 ? (kPairStages - 1) * MAT : buf - MAT; };
    auto move = [&](int tile) {
        window = 8 * tile & ~63;
        const int page = next;
        address = units.address(window + lane, page, bad);
        next = units.page_of(window + 64 + lane);
        if (wave == 0) {
            const int64_t at = scale_at(c, (unsigned)page >= (unsigned)c.num_pages ? 0 : page,
                                        (8 * units.seen(window + lane)) & units.pmask, bsh) + kvh;
            lds_dma_byte_at(__builtin_amdgcn_readfirstlane(bytes_at(tile)), (uint64_t)(c.k_scale + at));
            lds_dma_byte_at(__builtin_amdgcn_readfirstlane(bytes_at(tile) + 256), (uint64_t)(c.v_scale + at));
        }
    };
    // this wave's rows of a tile of K or V into its buffer; K goes ahead and moves the window
    auto stage = [&](auto which, int tile, uint32_t buf) {
        constexpr bool values = decltype(which)::value;
        if (tile < begin || tile >= end) return;
        const int k0 = kWideKeys * tile;
        if (!values && (8 * tile & ~63) != window) move(tile);
        const uint32_t dst = lds0 + (values ? kPairStages * MAT : 0) + buf, ln = lane_here(), dr = ln / 16, ds = ln % 16;
        auto rows_of = [&](auto all) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row0 = RPI * (wave + NW * i);
                const uint32_t row = row0 + dr, piece = 16u * (ds ^ (values ? pair_swizzle(row) : k_swizzle8<D>(row)));
                const int unit = 8 * tile + (row0 >> 3);
                uint32_t off = ((row0 & 7) + dr) * stride;
                // positions that no row sees are taken from the nearest one that some row sees
                if constexpr (!decltype(all)::value)
                    off = (uint32_t)(min(max(k0 + (int)row, t.lo), t.hi - 1) - 8 * units.seen(unit)) * stride;
                const uint64_t at = read_lane(address, unit - window) + (values ? v_from_k : 0);
                lds_dma16(__builtin_amdgcn_readfirstlane(dst + (uint32_t)row0 * D), off + piece, reinterpret_cast<const uint8_t*>(at));
            }
        };
        if (k0 >= t.lo && k0 + kWideKeys <= t.hi)
            rows_of(std::true_type());
        else
            rows_of(std::false_type());
    };
    // dims 32 j + 16 part + {0 .. 7, 8 .. 15} are this lane's of k-steps 2 j and 2 j + 1, as K's 16-byte reads have them
    h8 q[KS];
    const uint16_t* qrow = a.q + (int64_t)(s.q0 + token) * a.ld_q + (int64_t)(kvh * plan.group + head) * D + 16 * part;
#pragma unroll
    for (int k = 0; k < KS; ++k) q[k] = *reinterpret_cast<const h8*>(qrow + 32 * (k >> 1) + 8 * (k & 1));
    // The same where all of the tile is seen, a few instructions: the loop does it beside its products, where it is 2
    // to 4 % faster than at a turn's start.
    const int row0 = RPI * wave, unit0 = row0 >> 3;
    const uint32_t lane_off = ((row0 & 7) + (uint32_t)lane / 16) * stride;
    const uint32_t k_off = lane_off + 16u * ((uint32_t)lane % 16 ^ k_swizzle8<D>(row0 + lane / 16));
    const uint32_t v_off = lane_off + 16u * ((uint32_t)lane % 16 ^ pair_swizzle(row0 + lane / 16));
    static_assert(RPI * NW % 16 == 0, "one offset a lane for all of a wave's rows");
    auto stage_whole = [&](auto which, int tile, uint32_t buf) {
        constexpr bool values = decltype(which)::value;
        if (!values && (8 * tile & ~63) != window) move(tile);
        const uint32_t dst = lds0 + (values ? kPairStages * MAT : 0) + (uint32_t)row0 * D + buf;
        const int unit = 8 * tile - window + unit0;
#pragma unroll
        for (int i = 0; i < NI; ++i)
            lds_dma16(__builtin_amdgcn_readfirstlane(dst + (uint32_t)(RPI * NW * i) * D), values ? v_off : k_off,
                      reinterpret_cast<const uint8_t*>(read_lane(address, unit + RPI * NW / 8 * i) + (values ? v_from_k : 0)));
    };
    uint32_t buf = (uint32_t)(begin + 2) % kPairStages * MAT;    // of the tile before the first
    if (begin < end) {
        next = units.page_of((8 * begin & ~63) + lane);
        stage(std::false_type(), begin, after(buf));
        stage(std::true_type(), begin, after(buf));
        stage(std::false_type(), begin + 1, ahead_of(buf));
    }
    // the sign and a zero of the scale go to Q, as in wide_part
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
    const float scale = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
        q[k] = __builtin_bit_cast(h8, __builtin_bit_cast(u32x4, q[k]) ^ sign);
        if (a.scale == 0.0f) q[k] *= (_Float16)0;
    }
    // operand addresses: one base, and an xor for each piece
    const int krow = M * half + col;
    const uint32_t ka = lds0 + (uint32_t)krow * D + 16u * (uint32_t)(part ^ k_swizzle8<D>(krow));
    const int i16 = lane & 15, vr = 4 * part + ((i16 >> 1) & 3) + 8 * (i16 >> 3);
    const uint32_t va = lds0 + kPairStages * MAT + (uint32_t)vr * D +
                        16u * (uint32_t)((8 * half + ((lane >> 4) & 1)) ^ pair_swizzle(vr)) + 8u * (uint32_t)(i16 & 1);
    // a wave's weights and maxima of a tile
    const uint32_t weights_lane = weights0 + 16u * lane, tops_lane = tops0 + 4u * col;
    auto weights_at = [&](int wave, int tile) { return weights_lane + (uint32_t)((tile & 1) * NW + wave) * 2048; };
    auto top_at = [&](int wave, int tile) { return tops_lane + (uint32_t)((tile & 1) * NW + wave) * (4 * M); };
    f16v o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    // m: of the outputs, both waves'; own: of this wave's newest weights and of l
    float m = kNone, own = kNone, l = 0.0f, mul = scale;
    bool dirty = false;
    h8 p[4];                                     // the weights of this half's positions, and of the other's

    const uint32_t byte_lane = 4u * (4 * half + col / 8);
    // S^T of this wave's half of a tile
    auto scores = [&](int tile, uint32_t buf, f16v& x) {
        uint32_t kt = ka + buf;
        asm("" : "+v"(kt));
        const float ks = pow2_of(scale_byte(*(lds_int)(byte_lane + bytes_at(tile) + 4u * (8 * tile & 63))));
        auto codes = [&](int j) { return *(lds_u4)(kt ^ (32u * j)); };
        constexpr int AHEAD = 2;
        u32x4 w[AHEAD + 1];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) w[j] = codes(j);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = 0.0f;
#pragma unroll
        for (int j = 0; j < KS / 2; ++j) {
            if (j + AHEAD < KS / 2) w[(j + AHEAD) % (AHEAD + 1)] = codes(j + AHEAD);
            h8 lo, hi;
            values_of(w[j % (AHEAD + 1)], ks, lo, hi);
            x = G::mfma(lo, q[2 * j], x);
            x = G::mfma(hi, q[2 * j + 1], x);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Both halves' weights of a tile, under one maximum.
    auto meet = [&](int tile) {
        const uint32_t at = weights_at(wave ^ 1, tile);
#pragma unroll
        for (int i = 0; i < 2; ++i) p[2 + i] = *(lds_h8)(at + 1024u * i);
        const float other = *(lds_f)(top_at(wave ^ 1, tile));
        const float most = fmaxf(own, other);
        if (__ballot(most != m || most != own || most != other)) {
            const float f = __builtin_amdgcn_exp2f(m - most), g = __builtin_amdgcn_exp2f(own - most);
            // (in two factors: fp16 ends at 2^-24, and a weight of 2^15 times less than that may count)
            auto bring = [&](h8* q, float by) {
                const float some = ceilf(0.5f * by);
                const _Float16 a = (_Float16)__builtin_amdgcn_exp2f(some), b = (_Float16)__builtin_amdgcn_exp2f(by - some);
#pragma unroll
                for (int i = 0; i < 2; ++i) q[i] = q[i] * a * b;
            };
            bring(p, own - most);
            bring(p + 2, other - most);
            l *= g;
            m = own = most;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[i][e] *= f;
        }
    };
    // The softmax of x, a tile's scores, in two steps: the maximum, and the 2 n-th and next weight.
    auto maximum = [&](auto mask, int tile, f16v& x) {
        if constexpr (decltype(mask)::value) {
            const int ahead = pos - kWideKeys * tile - M * half - 4 * part, behind = a.window > 0 ? ahead - a.window : INT_MIN;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (G::key(e) > ahead || G::key(e) <= behind) x[e] = -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, x[e]);
        top = xor_butterfly<32, 32>(top, max_raw) * scale;
        const bool up = top > m + (kLag + kLift);
        own = up ? ceilf(top) - kLift : m;
        if (__ballot(up)) l *= up ? __builtin_amdgcn_exp2f(m - own) : 1.0f;
        // a score times the scale less the maximum in one fma; past 2^23, where the maximum was itself
        // rounded by a half and more, the product is rounded as it was
        const bool far = fabsf(own) >= 0x1p23f && own != kNone;
        mul = scale;
        if (__ballot(far)) {
            const float by = far ? scale : 1.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = __fmul_rn(x[e], by);
            mul = far ? 1.0f : scale;
        }
    };
    u32x4 w[2];
    float sum = 0.0f;                            // of a tile's weights
    auto weights = [&](int n, const f16v& x) {
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) f[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * n + i], mul, -own));
        w[n >> 2][n & 3] = __builtin_bit_cast(uint32_t, h2{(_Float16)f[0], (_Float16)f[1]});
        asm volatile("" : "+v"(w[n >> 2][n & 3]));               // here, not where it is used
        sum = (n == 0 ? 0.0f : sum) + (f[0] + f[1]);
        if (n == 7) l += sum;
    };
    auto give = [&](int tile) {
        const uint32_t at = weights_at(wave, tile);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            p[i] = __builtin_bit_cast(h8, w[i]);
            *(lds_h8w)(at + 1024u * i) = p[i];
        }
        if (part == 0) *(lds_f)(top_at(wave, tile)) = own;
    };
    // O^T += V^T P^T of a tile, 16 positions at a time, this wave's half first, their codes read a turn
    // ahead (the first ones by the caller); beside(n): what is done beside the n-th product
    i2 codes[2][NB];
    auto read_codes = [&](uint32_t buf, int f) {
        uint32_t vt = va + buf + (uint32_t)(M * (f < 2 ? half : 1 - half) + 16 * (f & 1)) * D;
        asm("" : "+v"(vt));
#pragma unroll
        for (int d = 0; d < NB; ++d) codes[f & 1][d] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2)(vt ^ (32u * d)));
    };
    auto product = [&](auto mask, int tile, uint32_t buf, auto beside) {
        // the exponents of 16 positions, as read
        auto bytes_of = [&](int f) {
            return *(lds_i2)(bytes_at(tile) + 256 + 4u * ((8 * tile & 63) + 4 * (f < 2 ? half : 1 - half) + 2 * (f & 1)));
        };
        i2 bytes = bytes_of(0);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const float vs[2] = {pow2_of(scale_byte(bytes[0])), pow2_of(scale_byte(bytes[1]))};
            if (f < 3) {
                read_codes(buf, f + 1);
                bytes = bytes_of(f + 1);
            }
            i2 (&now)[NB] = codes[f & 1];
            if constexpr (decltype(mask)::value) {
                // NaN among values that some rows do not see must not meet their zero weights: zeros
                // take its place, and the rows that see it get it at the end
                i2 nan = {0, 0};
#pragma unroll
                for (int d = 0; d < NB; ++d) nan |= (now[d] & 0x7f7f7f7f) + 0x01010101;
                if (__ballot(((nan[0] | nan[1]) & 0x80808080) != 0)) {
                    dirty = true;
#pragma unroll
                    for (int d = 0; d < NB; ++d) {
                        const i2 one = (((now[d] & 0x7f7f7f7f) + 0x01010101) >> 7) & 0x01010101;
                        now[d] &= ~((one << 8) - one);
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < NB; ++d) {
                const i2 k = now[d];
                const h8 v = join(__builtin_shufflevector(two_of<false>(k[0], vs[0]), two_of<true>(k[0], vs[0]), 0, 1, 2, 3),
                                  __builtin_shufflevector(two_of<false>(k[1], vs[1]), two_of<true>(k[1], vs[1]), 0, 1, 2, 3));
                o[d] = G::mfma(v, p[f], o[d]);
                beside(NB * f + d);
            }
        }
    };

    // the tiles that this pair's rows see, and among them those that all its rows see whole
    const int mine = active ? min(max(u.lo / kWideKeys, begin), end) : end;
    const int mine_end = active ? max(min((u.hi + kWideKeys - 1) / kWideKeys, end), mine) : end;
    const int behind = a.window > 0 ? max(u.last - a.window + kWideKeys, 0) / kWideKeys : 0;
    const int full = min(max(behind, mine), mine_end);
    const int full_end = min(max((u.first + 1) / kWideKeys, full), mine_end);
    f16v x;
    // A turn: a tile's product beside the scores and the softmax of the next one.  At its start this
    // wave's share of what is read has landed (all but what the turn before has asked for); past the
    // barrier everyone's has, the weights are there, and the buffers that are filled next have been read.
    auto start = [&](int tile) {
        if (tile + 2 < end)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NI) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();
        stage(std::true_type(), tile + 2, ahead_of(buf));
        stage(std::false_type(), tile + 3, buf);
    };
    const int seen_whole = min(end, t.hi / kWideKeys);           // (none of the loop's tiles begins in front of t.lo)
    int tile = begin - 1;
    while (true) {
        const int whole = full_end - 1;          // turns from full on have whole tiles on both sides
        const int stop = tile < full && full < whole ? full : end;
#pragma unroll 1
        for (; tile < stop; ++tile, buf = after(buf)) {
            start(tile);
            const bool more = tile + 1 >= mine && tile + 1 < mine_end;
            if (more) scores(tile + 1, after(buf), x);
            if (tile >= mine && tile < mine_end) {
                read_codes(buf, 0);
                meet(tile);
                product(std::true_type(), tile, buf, [](int) {});
            }
            if (more) {
                maximum(std::true_type(), tile + 1, x);
#pragma unroll
                for (int n = 0; n < 8; ++n) weights(n, x);
                give(tile + 1);
            }
        }
        if (tile >= end) break;
#pragma unroll 1
        for (; tile < whole; ++tile, buf = after(buf)) {
            const bool fast = tile + 3 < seen_whole;
            if (fast) {
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NI) : "memory");
                lds_barrier();
            } else {
                start(tile);
            }
            read_codes(buf, 0);
            meet(tile);
            // (a wave in its products goes before the SIMD's other one: 1 to 3 % of a launch)
            __builtin_amdgcn_s_setprio(2);
            scores(tile + 1, after(buf), x);
            __builtin_amdgcn_s_setprio(1);
            product(std::false_type(), tile, buf, [&](int n) {
                if (n == 0 && fast) stage_whole(std::true_type(), tile + 2, ahead_of(buf));
                if (n == 2 && fast) stage_whole(std::false_type(), tile + 3, buf);
                // (the scores have settled beside the first four)
                if (n == 3) maximum(std::false_type(), tile + 1, x);
                if (n >= 4 && n < 12) weights(n - 4, x);
                __builtin_amdgcn_sched_barrier(0);
            });
            __builtin_amdgcn_s_setprio(0);
            give(tile + 1);
        }
    }
    if (dirty) {
        // the NaN that were replaced, to the rows that see them: those of the tiles that were run masked
        const uint8_t* vc = c.v + kvh * c.head_stride + D / 2 * half + 4 * part;
#pragma unroll 1
        for (int k0 = kWideKeys * mine; k0 < kWideKeys * mine_end; ++k0) {
            if (k0 == kWideKeys * full) k0 = kWideKeys * max(full, full_end - 1);
            if (k0 >= kWideKeys * mine_end) break;
            if (k0 < t.lo || k0 >= t.hi) continue;
            const int page = units.table[k0 >> units.psh];
            if ((unsigned)page >= (unsigned)c.num_pages) continue;
            const uint8_t* row = vc + (int64_t)page * c.page_stride + (int64_t)(k0 & units.pmask) * c.row_stride;
            const bool seen = k0 <= pos && (a.window == 0 || k0 > pos - a.window);
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const uint32_t codes = *reinterpret_cast<const uint32_t*>(row + M * i + G::key(e));
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        o[i][e + n] = seen && ((codes >> (8 * n)) & 0x7f) == 0x7f ? NAN : o[i][e + n];
                }
        }
    }
    // both halves' sums
    l = xor_sum<32, 32>(l);
    if (bad) l = NAN;
    const uint32_t sum_at = sums0 + 4u * col;
    if (part == 0) *(lds_f)(sum_at + 4u * M * wave) = l;
    lds_barrier();
    l += *(lds_f)(sum_at + 4u * M * (wave ^ 1));
    if (pos == 0 || a.window == 1) l = (float)(_Float16)l;
    if (!active || w0 + col >= rows) return;
    const int d0 = D / 2 * half + 4 * part;
    if (s.parts > 1) {
        float* to = slot_of<ROWS, D>(plan.states, s, s.part, kvh, nkv);
        const int row = M * (wave >> 1) + col;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<f4*>(to + row * D + d0 + M * i + G::key(e)) = f4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
        if (half == 0 && part == 0) {
            to[ROWS * D + row] = m;
            to[ROWS * (D + 1) + row] = l;
        }
    } else {
        // (worked out again, not kept in registers over the loop)
        int row = w0 + col;
        asm("" : "+v"(row));
        const int tk = token_of(plan, row), hd = row - tk * plan.group;
        const float inv = s.kv - s.n + tk < 0 ? 0.0f : 1.0f / l;
        const int64_t at = (int64_t)(s.q0 + tk) * a.ld_out + (int64_t)(kvh * plan.group + hd) * D + d0;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                store4(a, at + M * i + G::key(e), f4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]} * inv);
    }
}

// ---- the launches -------------------------------------------------------------------------

// Waves and stages of the narrow part, waves of the wide one.  Two
// stages a wave, so that two and more workgroups share a CU: 48 requests of 60 to 16000 positions
// (head_dim 128, in the requests' order) 52.4 us, with three stages and one workgroup a CU 67; at 64 a third stage is even
// (47.7 and 48.1 us, 64 requests of 2000).  At 256 two waves, for the same reason: 256 requests
// of 600 138 us, with four waves 166.  HW: waves of a workgroup by itself on its CU, for a few hundred positions.
template <int D> struct Shape8;
template <> struct Shape8<64> { static constexpr int W = 4, S = 2, HW = 8, LW = 4, LS = 4, NW = 4; };
template <> struct Shape8<128> { static constexpr int W = 4, S = 2, HW = 8, LW = 4, LS = 2, NW = 4; };
template <> struct Shape8<256> { static constexpr int W = 2, S = 2, HW = 4, LW = 2, LS = 2, NW = 8; };
constexpr int kNarrowLeast8 = 4, kBesideLeast8 = 16, kWideLeast8 = 24;
constexpr int kFewWhole8 = 16, kManyWhole8 = 32, kWideWhole8 = 32;
template <int D>
constexpr int narrow8_lds(int w, int s) { return w * s * 2 * kNarrowKeys * D; }
template <int D>
constexpr int wide8_lds() { return D == 256 ? pair8_lds<D, Shape8<D>::NW>() : 4 * kWideKeys * 2 * D; }
template <int D>
constexpr int wide8_rows() { return 32 * Shape8<D>::NW / (D == 256 ? 2 : 1); }
static_assert(wide8_rows<64>() == kWideRows && wide8_rows<128>() == kWideRows && wide8_rows<256>() == kWideRows,
              "the workspace's tiles");

template <int D, int W>
__global__ __launch_bounds__(64 * W)
void rf_paged8_attn_narrow_kernel(const rf_paged_attention a, const rf_paged_cache8 c, const Plan plan) {
    constexpr int S = Shape8<D>::S;
    __shared__ __align__(1024) uint8_t lds[narrow8_lds<D>(W, S)];
    narrow8_part<D, W, S>(a, c, plan, (int)(blockIdx.x + blockIdx.y * gridDim.x), lds);
}

// Both kinds in one launch, the wide items first: their workgroups are the
// longer ones, and the narrow ones fill the CUs that they leave.
template <int D>
__global__ __launch_bounds__(64 * Shape8<D>::NW) __attribute__((amdgpu_waves_per_eu(2)))
void rf_paged8_attn_mixed_kernel(const rf_paged_attention a, const rf_paged_cache8 c, const Plan wide, const Plan narrow) {
    constexpr int LW = Shape8<D>::LW, LS = Shape8<D>::LS, NEED = narrow8_lds<D>(LW, LS);
    __shared__ __align__(1024) uint8_t lds[NEED > wide8_lds<D>() ? NEED : wide8_lds<D>()];
    const int item = (int)(blockIdx.x + blockIdx.y * gridDim.x);
    if (item < wide.items) {
        if constexpr (D == 256)
            pair8_part<D, Shape8<D>::NW>(a, c, wide, item, lds);
        else
            wide_part<D, Shape8<D>::NW, 32>(a, c, wide, item, lds);
    } else {
        if (threadIdx.x >= 64 * LW) return;      // whole waves, before any barrier
        narrow8_part<D, LW, LS>(a, c, narrow, item - wide.items, lds);
    }
}

template <int D>
__global__ __launch_bounds__(256) void rf_paged8_attn_join_kernel(const rf_paged_attention a, const rf_paged_cache8 c,
                                                                  const Plan wide, const Plan narrow, int wide_items) {
    __shared__ float weight[kJoinParts][kJoinRows];
    __shared__ f4 sums[256];
    const int item = blockIdx.x;
    if (item < wide_items)
        join_part<D, wide8_rows<D>(), kWideKeys>(a, c, wide, item, weight, sums);
    else
        join_part<D, kNarrowRows, kNarrowKeys>(a, c, narrow, item - wide_items, weight, sums);
}

}  // namespace rf

template <int D>
static void attn8_go(const rf_paged_attention& a, const rf_paged_cache8& c, hipStream_t stream) {
    using namespace rf;
    constexpr int ROWS = wide8_rows<D>();
    const int nkv = c.num_kv_heads, group = a.num_heads / nkv;
    const int64_t packed = (int64_t)a.rows * group, positions = (int64_t)a.max_blocks * c.page_size;
    const bool both = (int64_t)a.max_new * group > kNarrowRows;
    float* ws = static_cast<float*>(a.workspace);
    const auto inverse = [](int n) { return (uint32_t)(((1ll << 32) + n - 1) / n); };
    const uint32_t inv = packed * group < (1ll << 32) ? inverse(group) : 0;
    const int64_t some = std::min<int64_t>(a.num_seqs, a.rows);        // requests with rows
    const int64_t tiles = some * nkv;
    // Few tiles in a part a CU, more in nearly two, as the joins cost little beside the ragged
    // end then (head_dim 128): one request of 16000 positions 17.3 us at 256 parts and 18.9 at 400,
    // 20 of 4000 49.1 and 44.1, 48 of 60 to 16000 56.9, 52.4 and, at 512, 57.8.
    const int aim = tiles < 64 ? 256 : 400;
    const auto least = [&](int keys, int whole, int cut) { return positions <= whole * keys ? whole : cut; };
    // Two pieces a wave of a heavy workgroup, three from 64 tiles on: uncut by these, where there are no more tiles than
    // CUs.  us (head_dim 128), uncut by 8 waves / cut by 4: one request of 100 positions 5.7 / 5.3, of 300 6.8 / 7.4, of 500
    // 7.8 / 8.7, of 640 9.0 / 8.8, of 900 10.5 / 8.6; 8 of 640 9.7 / 11.2, 24 12.1 / 15.8, but 32 of 500 13.4 / 12.2.
    const int most = (tiles < 64 ? 2 : 3) * Shape8<D>::HW;
    const bool heavy = !both && tiles < 256 && positions > 6 * kNarrowKeys && positions <= most * kNarrowKeys;
    const int narrow_least = least(kNarrowKeys, heavy ? most : both || tiles >= 256 ? kManyWhole8 : kFewWhole8,
                                   both ? kBesideLeast8 : kNarrowLeast8);
    Plan narrow = {group, inv, 0, both ? kNarrowRows : INT_MAX, aim, narrow_least, inverse(aim), 0, ws};
    const int64_t wide_tiles = (packed / ROWS + std::min(some, packed / kNarrowRows)) * nkv;
    const int wide_aim = (int)std::max<int64_t>(wide_parts<D>() - wide_tiles / 4, wide_parts<D>() / 4);
    Plan wide = {group, inv, kNarrowRows, INT_MAX, wide_aim, least(kWideKeys, kWideWhole8, kWideLeast8), inverse(wide_aim), 0,
                 ws + narrow_bytes<D>() / sizeof(float)};
    // Items: every tile has a part, and there are at most as many parts more as are aimed at (each of
    // them a share long); no more either than the table's width gives room for.
    const auto items = [&](int64_t tiles, const Plan& p, int keys, int64_t* joins) {
        const int64_t most = std::max<int64_t>((positions + keys * p.least - 1) / (keys * p.least), 1);
        *joins = most > 1 ? std::min<int64_t>(tiles, p.parts) : 0;
        return (int)std::min(tiles + p.parts, tiles * most);
    };
    int64_t narrow_joins, wide_joins = 0;
    narrow.items = items((both ? some : packed / kNarrowRows + some) * nkv, narrow, kNarrowKeys, &narrow_joins);
    if (both) {
        wide.items = items(wide_tiles, wide, kWideKeys, &wide_joins);
        // (workgroups i and i + 8 share an XCD's L2, and items i and i + num_kv_heads their K and V)
        wide.items = (wide.items + 8 * nkv - 1) / (8 * nkv) * (8 * nkv);
    }
    const unsigned total = (unsigned)wide.items + (unsigned)narrow.items;
    const dim3 grid(std::min(total, 1u << 20), (total + (1u << 20) - 1) >> 20);
    if (both)
        hipLaunchKernelGGL(rf_paged8_attn_mixed_kernel<D>, grid, dim3(64 * Shape8<D>::NW), 0, stream, a, c, wide, narrow);
    else if (heavy)
        hipLaunchKernelGGL((rf_paged8_attn_narrow_kernel<D, Shape8<D>::HW>), grid, dim3(64 * Shape8<D>::HW), 0, stream, a, c, narrow);
    else
        hipLaunchKernelGGL((rf_paged8_attn_narrow_kernel<D, Shape8<D>::W>), grid, dim3(64 * Shape8<D>::W), 0, stream, a, c, narrow);
    const int wide_blocks = (int)wide_joins * (ROWS / kJoinRows);
    if (wide_joins + narrow_joins > 0)
        hipLaunchKernelGGL(rf_paged8_attn_join_kernel<D>, dim3((unsigned)(wide_blocks + narrow_joins)), dim3(256), 0,
                           stream, a, c, wide, narrow, wide_blocks);
}

extern "C" hipError_t rf_paged_attention8_launch(const rf_paged_attention* step, const rf_paged_cache8* cache,
                                                 hipStream_t stream) {
    if (step == nullptr || cache == nullptr) return hipErrorInvalidValue;
    rf_paged_attention a = *step;
    const rf_paged_cache8& c = *cache;
    if (!rf::cache8_ok(c) || !rf::attention_ok(a, c)) return hipErrorInvalidValue;
    if (a.rows == 0 || a.num_seqs == 0) return hipSuccess;
    if (!rf::attention_buffers_ok(a, c)) return hipErrorInvalidValue;
    if (a.window >= (int64_t)a.max_blocks * c.page_size) a.window = 0;     // reaches past every position
    switch (c.head_dim) {
    case 64: attn8_go<64>(a, c, stream); break;
    case 128: attn8_go<128>(a, c, stream); break;
    default: attn8_go<256>(a, c, stream); break;
    }
    return hipGetLastError();
}
