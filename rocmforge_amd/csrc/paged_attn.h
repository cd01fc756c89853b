// paged_attn.h -- what the attention over fp16 pages (paged_attn.hip) and over
// 8-bit pages (paged8_attn.hip) share: which part of which request a workgroup
// does, the kernel for pieces of prompt, and the join of parts.
//
// A request's rows are packed with the heads of a KV head's group: packed row
// r = token * group + head of the group, n * group of them a request and KV
// head, in tiles that share what they read of K and V.  Two kernels:
//   narrow  tiles of 16 packed rows, for requests of few rows (decode): each
//           wave streams its own pieces of K and V.  Memory-bound.
//   wide    tiles of 32 packed rows a wave, for pieces of prompt: the waves of
//           a workgroup share K and V.  MFMA-bound.
// Both compute S^T = K Q^T, so that a lane holds scores of one packed row and
// the weights in its accumulator registers are the B operand of O^T = V^T P^T
// as they are; V is transposed by its LDS reads.
//
// A tile's positions are cut into parts for several workgroups where that is
// needed to fill the chip or to even out long and short requests; a second
// kernel joins the parts' (m, l, O).  Lengths are in device memory, so every
// workgroup works its item out from them: a few loads and wave scans.
#pragma once
#include <hip/hip_fp16.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "paged8.h"
#include "paged_common.h"
#include "qk_common.h"

namespace rf {


typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) const h8* lds_h8;
typedef __attribute__((address_space(3))) s4* lds_s4;
typedef __attribute__((address_space(3))) const h4* lds_h4;
typedef __attribute__((address_space(3))) h8* lds_h8w;
typedef __attribute__((address_space(1))) const u32x4* global_u4;

constexpr float kNone = -3.0e+38f;               // the maximum of no scores
constexpr float kLog2e = 1.4426950408889634f;
// A row's maximum is left behind until a score passes it by more than 2^8: most
// tiles then rescale nothing.  Weights reach 256 (fp16 ends at 65504), and since
// the sum is of the rounded weights, a row of one key still has it exactly (heads of 256
// over 8-bit pages, whose sum is not, see to that by themselves).  Each row renews its own:
// were a wave's rows renewed together, keys that only some of them see would enter the
// others' roundings.
constexpr float kLag = 8.0f;
// Over 8-bit pages a row's maximum, as it is kept, is 2^7 below its largest score, so that weights reach 2^15, have
// their 11 bits down to 2^-21 and count down to 2^-32 of the largest.  A tile's are added up before they join the sum:
// what 100000 keys have beside one that leads by e^17 counts.
constexpr float kLift = 7.0f;

constexpr int kNarrowRows = 16, kNarrowKeys = 32;
constexpr int kWideKeys = 64;
constexpr int kNarrowParts = 512;                // the most narrow parts that are aimed at
// ---- which part of which request a workgroup does ---------------------------------------

struct Share {
    int b, q0, n, kv;            // the request, its first row, rows and positions
    int tiles, tile;             // of its packed rows
    int parts, part;             // of the tile's positions
    int slot;                    // workspace slot of part 0 of tile 0 (per KV head; parts > 1)
};

// What the host knows of a launch.
struct Plan {
    int group;
    uint32_t group_inv;          // 2^32 / group rounded up where r / group is the high word of r group_inv, else 0
    int from_rows, to_rows;      // requests of from_rows < packed rows <= to_rows are this kernel's
    int parts, least;            // parts aimed at, and the least units of one
    uint32_t parts_inv;          // 2^32 / parts, rounded up
    int items;                   // at least as many as there are
    float* states;               // the parts'
};

__device__ __forceinline__ int token_of(const Plan& p, int r) {
    return p.group == 1 ? r : p.group_inv ? (int)__umulhi((uint32_t)r, p.group_inv) : r / p.group;
}

struct Request {
    int q0, n, kv, tiles, units;
};

template <int ROWS, int KEYS, class C>
__device__ __forceinline__ Request request_of(const rf_paged_attention& a, const C& c, const Plan& p, int b) {
    Request r = {0, 0, 0, 0, 0};
    if (b >= a.num_seqs) return r;
    r.q0 = min(max(a.q_start[b], 0), a.rows);
    r.n = max(min(a.q_start[b + 1], a.rows) - r.q0, 0);
    r.kv = (int)min((int64_t)max(a.kv_lens[b], 0), (int64_t)a.max_blocks * c.page_size);
    const int rows = r.n * p.group;
    if (rows <= p.from_rows || rows > p.to_rows) return r;
    r.tiles = (rows + ROWS - 1) / ROWS;
    // (a window's first tile of keys is entered in the middle)
    const int seen = a.window > 0 ? (int)min((int64_t)r.kv, (int64_t)a.window + ROWS / p.group + KEYS) : r.kv;
    r.units = (seen + KEYS - 1) / KEYS;
    return r;
}

// Units a part: total / parts.  A tile is cut only where it is longer, so at most
// twice as many parts are written.  (In integers: the join has to come to the same.)
template <int ROWS, int KEYS, class C>
__device__ __forceinline__ int share_of(const rf_paged_attention& a, const C& c, const Plan& p,
                                        const Request& first) {
    const int lane = threadIdx.x & 63;
    int64_t mine = (int64_t)first.tiles * first.units;
    for (int b0 = 64; b0 < a.num_seqs; b0 += 64) {
        const Request r = request_of<ROWS, KEYS>(a, c, p, b0 + lane);
        mine += (int64_t)r.tiles * r.units;
    }
    const int64_t total = (((int64_t)wave_total((int)(mine >> 24)) << 24) + wave_total((int)(mine & 0xffffff))) *
                          c.num_kv_heads;
    // (rounded up; in 32 bits, in steps of 2^20 where the sum has more)
    const int sh = total >> 31 ? 20 : 0;
    const uint32_t steps = (uint32_t)((total + (1 << sh) - 1) >> sh), each = __umulhi(max(steps, 1u) - 1, p.parts_inv) + 1;
    return (int)min(max((int64_t)each << sh, (int64_t)p.least), (int64_t)1 << 30);
}

// Item j: the j-th (part, tile) over the requests, or (merge) the j-th tile of
// more than one part.  False where there is none.  Wave-uniform.
template <int ROWS, int KEYS, class C>
__device__ __forceinline__ bool find_share(const rf_paged_attention& a, const C& c, const Plan& p, int j,
                                           bool merge, Share& s) {
    const int lane = threadIdx.x & 63;
    const Request first = request_of<ROWS, KEYS>(a, c, p, lane);
    const int share = share_of<ROWS, KEYS>(a, c, p, first);
    int items_before = 0, slots_before = 0;
    for (int b0 = 0; b0 < a.num_seqs; b0 += 64) {
        const Request r = b0 == 0 ? first : request_of<ROWS, KEYS>(a, c, p, b0 + lane);
        const int parts = max((int)(((unsigned)r.units + share - 1) / (unsigned)share), 1);
        const int items = merge ? (parts > 1 ? r.tiles : 0) : r.tiles * parts;
        const int slots = parts > 1 ? r.tiles * parts : 0;
        const int items_end = items_before + wave_scan(items), slots_end = slots_before + wave_scan(slots);
        const uint64_t past = __ballot(items_end > j);
        if (past) {
            const int l = __builtin_ctzll(past);
            auto get = [l](int v) { return __builtin_amdgcn_readlane(v, l); };
            s.b = b0 + l;
            s.q0 = get(r.q0);
            s.n = get(r.n);
            s.kv = get(r.kv);
            s.tiles = get(r.tiles);
            s.parts = get(parts);
            s.slot = get(slots_end - slots);
            const int at = j - get(items_end - items);
            // the tiles of a part one after the other (they share K and V), the longest first
            s.part = at / s.tiles;
            s.tile = s.tiles - 1 - (at - s.part * s.tiles);
            return true;
        }
        items_before = __builtin_amdgcn_readlane(items_end, 63);
        slots_before = __builtin_amdgcn_readlane(slots_end, 63);
    }
    return false;
}

// Positions of a tile's packed rows [r0, r1]: keys [lo, hi) are seen by some of them.
struct Span {
    int first, last;             // positions of the first and the last row
    int lo, hi;
};
__device__ __forceinline__ Span span_of(const Plan& p, const Share& s, int r0, int r1, int window) {
    Span t;
    t.first = s.kv - s.n + token_of(p, r0);
    t.last = s.kv - s.n + token_of(p, r1);
    t.hi = max(t.last + 1, 0);
    t.lo = window > 0 ? (int)max((int64_t)t.first - window + 1, (int64_t)0) : 0;
    return t;
}

// The workspace slot of a part: O [ROWS][D], then m [ROWS], l [ROWS].
template <int ROWS, int D>
__device__ __forceinline__ float* slot_of(float* ws, const Share& s, int part, int kvh, int nkv) {
    const int64_t i = (int64_t)(s.slot + part * s.tiles + s.tile) * nkv + kvh;
    return ws + i * (ROWS * (D + 2));
}

__device__ __forceinline__ void store4(const rf_paged_attention& a, int64_t at, f4 v) {
    if (a.out_f32) {
        *reinterpret_cast<f4*>(static_cast<float*>(a.out) + at) = v;
    } else {
        const uint32_t x = (uint32_t)f16_bits_rn(v[0]) | ((uint32_t)f16_bits_rn(v[1]) << 16);
        const uint32_t y = (uint32_t)f16_bits_rn(v[2]) | ((uint32_t)f16_bits_rn(v[3]) << 16);
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + at) = u32x2{x, y};
    }
}

// Rows of K and V in LDS lie as in memory; a row's 16-byte pieces are permuted
// so that no read of the MFMA operands meets a bank twice: K's 16 lanes read one
// piece of 16 rows, V's transposing reads 32 (or 64) bytes of 4 (or 8) rows.
template <int D>
__device__ __forceinline__ int k_swizzle(int row) { return D == 64 ? (row >> 1) & 7 : row & 15; }
template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
    return (D == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3)) ^ (2 * ((row >> 2) & 1));
}

// LDS DMA of a group of rows: lanes a row, rows an instruction.
template <int D>
struct Dma {
    static constexpr int LPR = D / 8, RPI = 64 / LPR;
};

// Where K's rows of a request lie, by units of 8 positions (no page is smaller):
// a lane holds the address of one unit, so that a group of rows costs two lane
// reads and no table lookup or product.  lo, hi: the positions that are seen; units
// outside are taken from the nearest one inside.
template <class C>
struct Units {
    const int* table;
    decltype(C::k) k;
    int psh, pmask, unit_lo, unit_hi, num_pages;
    int64_t page_stride, row_stride;
    __device__ __forceinline__ Units(const rf_paged_attention& a, const C& c, int b, int kvh, int lo, int hi)
        : table(a.block_tables + (int64_t)b * a.max_blocks), k(c.k + kvh * c.head_stride), psh(__ffs(c.page_size) - 1),
          pmask(c.page_size - 1), unit_lo(lo >> 3), unit_hi((hi - 1) >> 3), num_pages(c.num_pages),
          page_stride(c.page_stride), row_stride(c.row_stride) {}
    __device__ __forceinline__ int seen(int unit) const { return min(max(unit, unit_lo), unit_hi); }
    __device__ __forceinline__ int page_of(int unit) const { return table[(8 * seen(unit)) >> psh]; }
    // page: page_of(unit); one outside the cache is read as page 0, and reported
    __device__ __forceinline__ uint64_t address(int unit, int page, bool& bad) const {
        const bool out = (unsigned)page >= (unsigned)num_pages;
        bad = bad || __ballot(out) != 0;
        return reinterpret_cast<uint64_t>(k + (int64_t)(out ? 0 : page) * page_stride +
                                          (int64_t)((8 * seen(unit)) & pmask) * row_stride);
    }
};
__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane) |
           ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32);
}

// One LDS read of four keys of one dim: 16 lanes read 4 rows of 32 bytes (lane i
// row i / 4, 8-byte piece i % 4) and receive dim i's four keys.
__device__ __forceinline__ h4 read_tr(uint32_t at) {
    return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)at));
}

__device__ __forceinline__ h8 join(h4 a, h4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// 16 codes times a power of two, as two MFMA operands
__device__ __forceinline__ void values_of(u32x4 w, float scale, h8& lo, h8& hi) {
    auto four = [&](uint32_t a, uint32_t b) {
        return join(__builtin_shufflevector(two_of<false>(a, scale), two_of<true>(a, scale), 0, 1, 2, 3),
                    __builtin_shufflevector(two_of<false>(b, scale), two_of<true>(b, scale), 0, 1, 2, 3));
    };
    lo = four(w[0], w[1]);
    hi = four(w[2], w[3]);
}

// l + the eight weights, products with one in fp32.
__device__ __forceinline__ float sum8(h8 p, float l) {
    const h2 one = {1, 1};
#pragma unroll
    for (int i = 0; i < 4; ++i) l = __builtin_amdgcn_fdot2(h2{p[2 * i], p[2 * i + 1]}, one, l, false);
    return l;
}

// Whether any of the values is an infinity or NaN: 0 * x is then not 0.
struct Finite {
    h8 acc = {0, 0, 0, 0, 0, 0, 0, 0};
    __device__ __forceinline__ void take(h8 v) { acc += v * (_Float16)0; }
    __device__ __forceinline__ bool all() const {
        bool ok = true;
#pragma unroll
        for (int i = 0; i < 8; ++i) ok = ok && acc[i] == (_Float16)0;
        return __ballot(!ok) == 0;
    }
};
// The value, or a finite one in the place of an infinity or NaN.
template <class V>
__device__ __forceinline__ V finite_of(V v) {
    const V most = (V)(_Float16)65504.0f;
    return __builtin_elementwise_min(__builtin_elementwise_max(v, -most), most);
}

// ---- pieces of prompt -------------------------------------------------------------------
//
// NW waves of M packed rows each over tiles of 64 positions, K and V by LDS
// DMA, double buffered, one barrier a tile.  The scores of a tile are computed
// beside the weights of the one before (MFMA beside exp), so K runs a tile ahead.
// M = 32 where a wave's queries and outputs fit its registers (head_dim 64 and
// 128); at 256 they would take 192 of them, and M = 16 has two waves a SIMD: a
// step of three windowed prompts 71 us, with 32 rows a wave, one wave a SIMD and
// outputs in accumulation registers 79.
// Bound at head_dim 128 by MFMA, softmax VALU and LDS reads, each about half of
// the time busy and overlapping across two waves a SIMD: a fresh prompt of 8192
// (32 heads on 8) 543 to 593 us, 930 to 1010 TFLOP/s where a large product reaches
// 1160; 512 tokens behind 15700 153 to 164 us.  At 256 by LDS reads (4096 clocks
// a CU and tile beside 2048 of MFMA): 390 TFLOP/s.

// The two MFMA shapes.  M packed rows a wave; acc: a block of scores or outputs, whose
// element e belongs to key (or dim) key(e) + 4 (lane / M) of it; DK dims a step of the scores,
// PK keys a step of the product.
template <int M>
struct Geo;
template <>
struct Geo<32> {
    typedef f16v acc;
    static constexpr int E = 16, DK = 16, PK = 16;
    static __device__ __forceinline__ constexpr int key(int e) { return 8 * (e >> 2) + (e & 3); }
    static __device__ __forceinline__ acc mfma(h8 a, h8 b, acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Geo<16> {
    typedef f4 acc;
    static constexpr int E = 4, DK = 32, PK = 32;
    static __device__ __forceinline__ constexpr int key(int e) { return e; }
    static __device__ __forceinline__ acc mfma(h8 a, h8 b, acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

template <int D, int NW, int M, class C>
__device__ __forceinline__ void wide_part(const rf_paged_attention& a, const C& c, const Plan& plan,
                                          int item, uint8_t* lds) {
    constexpr int ROWB = 2 * D, MAT = kWideKeys * ROWB, ROWS = M * NW;
    constexpr int LPR = Dma<D>::LPR, RPI = Dma<D>::RPI, NI = kWideKeys / (RPI * NW);   // a wave's instructions a tile
    typedef Geo<M> G;
    typedef typename G::acc Acc;
    constexpr int KS = D / G::DK, NB = D / M, XB = kWideKeys / M, E = G::E, XE = XB * E;
    constexpr bool BESIDE = M == 32;             // the next tile's scores beside a tile's weights
    constexpr bool CODES = std::is_same_v<C, rf_paged_cache8>;
    constexpr float LIFT = CODES ? kLift : 0.0f;
    static_assert(NI >= 1, "every wave has rows to fetch");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane % M, part = lane / M;   // a lane's packed row, and which keys or dims of it it has
    const int nkv = c.num_kv_heads;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const int dr = lane / LPR, ds = lane % LPR;

    Share s;
    const int kvh = item % nkv;
    if (!find_share<ROWS, kWideKeys>(a, c, plan, item / nkv, false, s)) return;
    const int rows = s.n * plan.group, r0 = ROWS * s.tile;
    const Span t = span_of(plan, s, r0, min(r0 + ROWS, rows) - 1, a.window);
    const int w0 = r0 + M * wave;
    const bool active = w0 < rows;
    const Span u = span_of(plan, s, min(w0, rows - 1), min(w0 + M, rows) - 1, a.window);
    const int p0 = t.lo / kWideKeys, p1 = (t.hi + kWideKeys - 1) / kWideKeys;
    const int each = (max(p1 - p0, 0) + s.parts - 1) / s.parts;
    const int begin = p0 + s.part * each, end = min(begin + each, p1);
    const int r = min(w0 + col, rows - 1), token = token_of(plan, r), head = r - token * plan.group;
    const int pos = s.kv - s.n + token;
    // the addresses of 64 units, and the pages of the next 64
    const Units<C> units(a, c, s.b, kvh, t.lo, t.hi);
    bool bad = false;
    int next = 0, window = -1;
    uint64_t address = 0;
    const uint64_t v_from_k = (uint64_t)c.v - (uint64_t)c.k;
    const uint32_t stride = (uint32_t)(2 * c.row_stride);
    const int wave_row = RPI * wave;
    // (a wave's groups of rows are a multiple of 16 apart: the same row of a unit, the same swizzle)
    static_assert(RPI * NW % 16 == 0, "one piece a lane for all of them");
    const uint32_t lane_row = (uint32_t)((wave_row & 7) + dr) * stride;
    const uint32_t k_piece = 16u * (uint32_t)(ds ^ k_swizzle<D>(wave_row + dr));
    const uint32_t v_piece = 16u * (uint32_t)(ds ^ v_swizzle<D>(wave_row + dr));
    // this wave's rows of a tile of K or V into its buffer; K goes first and moves the window
    [[maybe_unused]] auto stage = [&](auto which, int tile) {
        constexpr bool values = decltype(which)::value;
        if (tile < begin || tile >= end) return;
        const int k0 = kWideKeys * tile;
        if (!values && (8 * tile & ~63) != window) {
            window = 8 * tile & ~63;
            address = units.address(window + lane, next, bad);
            next = units.page_of(window + 64 + lane);
        }
        const uint32_t dst = lds0 + (values ? 2 * MAT : 0) + (uint32_t)(tile & 1) * MAT + 1024u * wave;
        const int u0 = 8 * tile - window;
        auto fetch = [&](auto all) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = wave_row + RPI * NW * i;
                int unit = u0 + (row >> 3);
                uint32_t off = lane_row + (values ? v_piece : k_piece);
                if constexpr (!decltype(all)::value) {
                    // positions that no row sees are taken from the nearest one that some row sees
                    unit = units.seen(unit + window);
                    off = (uint32_t)(min(max(k0 + row + dr, t.lo), t.hi - 1) - 8 * unit) * stride +
                          (values ? v_piece : k_piece);
                    unit -= window;
                }
                const uint64_t at = read_lane(address, unit) + (values ? v_from_k : 0);
                lds_dma16(__builtin_amdgcn_readfirstlane(dst + 1024u * NW * i), off, reinterpret_cast<const uint8_t*>(at));
            }
        };
        if (k0 >= t.lo && k0 + kWideKeys <= t.hi)
            fetch(std::true_type());
        else
            fetch(std::false_type());
    };
    // Codes come through registers and are written to LDS as the fp16 values that they stand for, each once:
    // fetch a tile's (this wave's share), put them a tile later.
    constexpr int LPC = D / 16, RPC = 64 / LPC, NC = CODES ? kWideKeys / (RPC * NW) : 1;
    static_assert(!CODES || (NC >= 1 && BESIDE), "every wave has rows to fetch, and K runs a tile ahead");
    u32x4 k_codes[NC], v_codes[NC];
    int scales = 0, scales_before = 0;           // a unit's exponents, V's << 8: of this window and of the one before
    const int cr = lane / LPC, cp = lane % LPC;
    // the unit of the wave's i-th group of rows, from the tile's first on; for heads of 64 of its first half
    auto group_unit = [&](int i) { return RPC * (wave + NW * i) >> 3; };
    auto fetch = [&](auto which, int tile) {
        constexpr bool values = decltype(which)::value;
        if constexpr (CODES) {
            if (tile < begin || tile >= end) return;
            if (!values && (8 * tile & ~63) != window) {
                window = 8 * tile & ~63;
                const int page = next;
                address = units.address(window + lane, page, bad);
                next = units.page_of(window + 64 + lane);
                const int64_t at = scale_at(c, (unsigned)page >= (unsigned)c.num_pages ? 0 : page,
                                            (8 * units.seen(window + lane)) & units.pmask, block_shift(c)) + kvh;
                scales_before = scales;
                scales = c.k_scale[at] | (c.v_scale[at] << 8);
            }
            const int u0 = 8 * tile - window, k0 = kWideKeys * tile;
            const bool whole = k0 >= t.lo && k0 + kWideKeys <= t.hi;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int row = RPC * (wave + NW * i) + cr;
                // positions that no row sees are taken from the nearest one that some row sees
                const int key = whole ? k0 + row : min(max(k0 + row, t.lo), t.hi - 1);
                int unit = 8 * tile + group_unit(i);
                uint64_t at;
                if constexpr (RPC > 8) {         // two units
                    const uint64_t lo = read_lane(address, u0 + group_unit(i)), hi = read_lane(address, u0 + group_unit(i) + 1);
                    unit = units.seen(unit + (lane >> 5));
                    at = lane < 32 ? lo : hi;
                } else {
                    unit = units.seen(unit);
                    at = read_lane(address, unit - window);
                }
                at += (uint64_t)((uint32_t)(key - 8 * unit) * (uint32_t)c.row_stride + 16u * (uint32_t)cp);
                (values ? v_codes : k_codes)[i] = *(global_u4)(at + (values ? v_from_k : 0));
            }
        }
    };
    auto put = [&](auto which, int tile) {
        constexpr bool values = decltype(which)::value;
        if constexpr (CODES) {
            if (tile < begin || tile >= end) return;
            const int w0 = 8 * tile & ~63, held = w0 == window ? scales : scales_before;
            const uint32_t dst = lds0 + (values ? 2 * MAT : 0) + (uint32_t)(tile & 1) * MAT;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int unit = 8 * tile + group_unit(i), row = RPC * (wave + NW * i) + cr;
                int byte = __builtin_amdgcn_readlane(held, units.seen(unit) - w0);
                if constexpr (RPC > 8) byte = lane < 32 ? byte : __builtin_amdgcn_readlane(held, units.seen(unit + 1) - w0);
                h8 lo, hi;
                values_of((values ? v_codes : k_codes)[i], pow2_of(scale_byte((values ? byte >> 8 : byte) & 0xff)), lo, hi);
                const uint32_t to = dst + (uint32_t)row * ROWB +
                                    16u * (uint32_t)((2 * cp) ^ (values ? v_swizzle<D>(row) : k_swizzle<D>(row)));
                *(lds_h8w)(to) = lo;
                *(lds_h8w)(to ^ 16u) = hi;
            }
        }
    };
    if (begin < end) {
        next = units.page_of((8 * begin & ~63) + lane);
        if constexpr (CODES) {
            fetch(std::false_type(), begin);
            fetch(std::true_type(), begin);
            put(std::false_type(), begin);
            put(std::true_type(), begin);
            fetch(std::false_type(), begin + 1);
            put(std::false_type(), begin + 1);
            fetch(std::true_type(), begin + 1);
            fetch(std::false_type(), begin + 2);
        } else {
            stage(std::false_type(), begin);
            stage(std::true_type(), begin);
            if constexpr (BESIDE) stage(std::false_type(), begin + 1);
        }
    }
    // a negative scale moves its sign to Q (exact), so that the largest S has the largest weight; a
    // scale of zero goes to Q whole, so that what is infinite in Q or K gives NaN
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
    const float scale = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);
    h8 q[KS];
    const uint16_t* qrow = a.q + (int64_t)(s.q0 + token) * a.ld_q + (int64_t)(kvh * plan.group + head) * D + 8 * part;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
        q[k] = __builtin_bit_cast(h8, *reinterpret_cast<const u32x4*>(qrow + G::DK * k) ^ sign);
        if (a.scale == 0.0f) q[k] *= (_Float16)0;
    }
    // operand addresses: one base, and an xor for each k-step or block of dims
    const int i16 = lane & 15, vr = 4 * part + (i16 >> 2);
    const uint32_t ka = lds0 + (uint32_t)col * ROWB + 16u * (uint32_t)(part ^ k_swizzle<D>(col));
    const uint32_t va = lds0 + 2 * MAT + (uint32_t)vr * ROWB +
                        16u * (uint32_t)(((M == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((i16 >> 1) & 1)) ^ v_swizzle<D>(vr)) +
                        8u * (uint32_t)(i16 & 1);
    Acc o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) o[i][e] = 0.0f;
    float m = kNone, l = 0.0f;
    bool far = false, dirty = false;

    // S^T of a tile; beside(n): what is done beside the n-th two of its products
    auto scores = [&](int tile, Acc (&y)[XB], auto beside) {
        // (opaque, so that a tile's addresses are not kept in registers over the loop)
        uint32_t kt = ka + (uint32_t)(tile & 1) * MAT;
        asm("" : "+v"(kt));
        auto k_frag = [&](int k, int b) { return *(lds_h8)((kt ^ (2u * G::DK * k)) + (uint32_t)(M * b) * ROWB); };
#pragma unroll
        for (int b = 0; b < XB; ++b)
#pragma unroll
            for (int e = 0; e < E; ++e) y[b][e] = 0.0f;
        // two blocks at a time, their operands two k-steps ahead
        constexpr int AHEAD = 2;
#pragma unroll
        for (int b0 = 0; b0 < XB; b0 += 2) {
            h8 kf[AHEAD + 1][2];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
#pragma unroll
                for (int b = 0; b < 2; ++b) kf[k][b] = k_frag(k, b0 + b);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                if (k + AHEAD < KS)
#pragma unroll
                    for (int b = 0; b < 2; ++b) kf[(k + AHEAD) % (AHEAD + 1)][b] = k_frag(k + AHEAD, b0 + b);
#pragma unroll
                for (int b = 0; b < 2; ++b) y[b0 + b] = G::mfma(kf[k % (AHEAD + 1)][b], q[k], y[b0 + b]);
                beside(b0 / 2 * KS + k);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // The softmax of x, a tile's scores, beside the next tile's, and its product with V
    auto step = [&](auto mask, int tile, Acc (&x)[XB], Acc (&y)[BESIDE ? XB : 1]) {
        constexpr bool masked = decltype(mask)::value;
        const int k0 = kWideKeys * tile;
        if constexpr (!BESIDE) scores(tile, x, [](int) {});
        uint32_t vt = va + (uint32_t)(tile & 1) * MAT;
        asm("" : "+v"(vt));
        // V^T (k-step j, block of dims i): the lane takes its dim's keys in the order in which the
        // weights' registers hold them, PK j + 4 part + {0 .. 3, PK / 2 ..}
        auto v_frag = [&](int j, int i) {
            const uint32_t v = (vt ^ (2u * M * i)) + (uint32_t)(G::PK * j) * ROWB;
            return join(read_tr(v), read_tr(v + (uint32_t)(G::PK / 2) * ROWB));
        };
        if constexpr (masked) {
            const int ahead = pos - k0 - 4 * part, behind = a.window > 0 ? ahead - a.window : INT_MIN;
#pragma unroll
            for (int b = 0; b < XB; ++b)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int key = M * b + G::key(e);       // less k0 + 4 part
                    if (key > ahead || key <= behind) x[b][e] = -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < XB; ++b)
#pragma unroll
            for (int e = 0; e < E; ++e) top = fmaxf(top, x[b][e]);
        top = xor_butterfly<32, M>(top, max_raw) * scale;
        // exp(x - m) as 2^(x scale - m), one fma: m is a rounded product and the fma's is not, so
        // a row's weights are off by one common factor of 2^(half a step of m).  Far from zero
        // (2^7) scores are rounded as m is, lest the factor leave fp16's range.
        const bool up = top > m + (kLag + LIFT);
        float mul = scale;
        if (__ballot(up || far)) {
            const float f = up ? __builtin_amdgcn_exp2f(m - (top - LIFT)) : 1.0f;
            m = up ? top - LIFT : m;
            l *= f;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) o[i][e] *= f;
            far = fabsf(m) >= 128.0f && m != kNone;
            if (__ballot(far)) {
                const float by = far ? scale : 1.0f;
#pragma unroll
                for (int b = 0; b < XB; ++b)
#pragma unroll
                    for (int e = 0; e < E; ++e) x[b][e] = __fmul_rn(x[b][e], by);
                mul = far ? 1.0f : scale;
            }
        }
        // (past the last tile of K the scores are of what its buffer holds, and are not used)
        constexpr int STEPS = XE / 8;            // of the product
        u32x4 w[STEPS];                          // the weights, two in a register
        // V's operands, in fours: those of the first products are read beside the scores, the others
        // one or two fours ahead
        constexpr int FOURS = STEPS * NB / 4, AHEAD = FOURS < 2 ? FOURS : M == 32 ? 2 : 1;
        h8 v[AHEAD + 1][4];
        auto read_four = [&](int f) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[f % (AHEAD + 1)][i] = v_frag((4 * f + i) / NB, (4 * f + i) % NB);
        };
        constexpr int TWOS = KS * XB / 2;
        auto weights = [&](int two) {
#pragma unroll
            for (int n = 0; n < XE; n += 2) {
                if (n / 2 * TWOS / (XE / 2) != two) continue;
                float f[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    f[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[n / E][n % E + i], mul, -m));
                w[n >> 3][(n >> 1) & 3] = __builtin_bit_cast(uint32_t, h2{(_Float16)f[0], (_Float16)f[1]});
                asm volatile("" : "+v"(w[n >> 3][(n >> 1) & 3]));        // here, not where it is used
            }
#pragma unroll
            for (int f = 0; f < AHEAD; ++f)
                if (two == TWOS - 1 - AHEAD + f) read_four(f);
        };
        if constexpr (BESIDE) {
            scores(tile + 1, y, weights);
        } else {
#pragma unroll
            for (int two = 0; two < TWOS; ++two) weights(two);
        }
        h8 p[STEPS];
        float sum = CODES ? 0.0f : l;
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
            p[j] = __builtin_bit_cast(h8, w[j]);
            sum = sum8(p[j], sum);
        }
        l = CODES ? l + sum : sum;
        // infinities and NaN among values that some rows do not see must not meet their zero
        // weights: finite ones take their place, and the rows that see them get them at the end
        Finite fin;
#pragma unroll
        for (int f = 0; f < FOURS; ++f) {
            if (f + AHEAD < FOURS) read_four(f + AHEAD);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = (4 * f + i) / NB, d = (4 * f + i) % NB;
                h8 b = v[f % (AHEAD + 1)][i];
                if constexpr (masked) {
                    fin.take(b);
                    b = finite_of(b);
                }
                o[d] = G::mfma(b, p[j], o[d]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (masked) dirty = dirty || !fin.all();
    };

    // (With the next scores beside, K runs a tile ahead of V.)  At a tile's start this wave's share
    // of what its step reads has landed; past the barrier everyone's has, and the buffers
    // that are filled next have been read.
    auto advance = [&](int tile) {
        if constexpr (CODES) {
            lds_barrier();                       // (this wave's values are written, and the next ones still on their way)
            if (tile < begin) return;
            put(std::true_type(), tile + 1);
            put(std::false_type(), tile + 2);
            fetch(std::true_type(), tile + 2);
            fetch(std::false_type(), tile + 3);
            return;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();
        if (tile < begin) return;
        if constexpr (!BESIDE) stage(std::false_type(), tile + 1);
        stage(std::true_type(), tile + 1);
        if constexpr (BESIDE) stage(std::false_type(), tile + 2);
    };
    // the tiles that this wave's rows see, and among them those that all its rows see whole
    const int mine = active ? min(max(u.lo / kWideKeys, begin), end) : end;
    const int mine_end = active ? max(min((u.hi + kWideKeys - 1) / kWideKeys, end), mine) : end;
    const int behind = a.window > 0 ? max(u.last - a.window + kWideKeys, 0) / kWideKeys : 0;
    const int full = min(max(behind, mine), mine_end);
    const int full_end = min(max((u.first + 1) >> 6, full), mine_end);
    int tile = begin - 1;
#pragma unroll 1
    for (; tile < mine - 1; ++tile) advance(tile);
    if (mine < mine_end) {
        Acc x[XB], y[BESIDE ? XB : 1];
        advance(tile++);
        if constexpr (BESIDE) scores(mine, x, [](int) {});
        // (whole tiles in pairs, so that x and y change places without copies)
        auto run = [&](auto mask, int to) {
            constexpr bool pairs = !decltype(mask)::value;
#pragma unroll 1
            for (; tile < to; ++tile) {
                advance(tile);
                step(mask, tile, x, y);
                if constexpr (BESIDE) {
                    if (pairs && tile + 1 < to) {
                        advance(++tile);
                        step(mask, tile, y, x);
                    } else {
#pragma unroll
                        for (int b = 0; b < XB; ++b) x[b] = y[b];
                    }
                }
            }
        };
        run(std::true_type(), full);
        run(std::false_type(), full_end);
        run(std::true_type(), mine_end);
    }
#pragma unroll 1
    for (; tile < end; ++tile) advance(tile);
    if (dirty) {
        // the values that were replaced, to the rows that see them: those of the tiles that were run masked
        const int psh = units.psh, pmask = units.pmask;
        const int* table = units.table;
        const auto* vc = c.v + kvh * c.head_stride;
#pragma unroll 1
        for (int k0 = kWideKeys * mine; k0 < kWideKeys * mine_end; ++k0) {
            if (k0 == kWideKeys * full) k0 = kWideKeys * full_end;
            if (k0 >= kWideKeys * mine_end) break;
            if (k0 < t.lo || k0 >= t.hi) continue;
            const int page = table[k0 >> psh];
            if ((unsigned)page >= (unsigned)c.num_pages) continue;
            const auto* row = vc + (int64_t)page * c.page_stride + (int64_t)(k0 & pmask) * c.row_stride + 4 * part;
            const bool seen = k0 <= pos && (a.window == 0 || k0 > pos - a.window);
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    if constexpr (CODES) {       // (NaN is all that a code can stand for beside what is finite)
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(row + M * i + G::key(e));
#pragma unroll
                        for (int n = 0; n < 4; ++n)
                            o[i][e + n] = seen && ((w >> (8 * n)) & 0x7f) == 0x7f ? NAN : o[i][e + n];
                    } else {
                        const h4 w = *reinterpret_cast<const h4*>(row + M * i + G::key(e)), f = finite_of(w);
#pragma unroll
                        for (int n = 0; n < 4; ++n)
                            o[i][e + n] = seen ? o[i][e + n] + ((float)w[n] - (float)f[n]) : o[i][e + n];
                    }
                }
        }
    }
    if (active && w0 + col < rows) {
        l = xor_sum<32, M>(l);
        if (bad) l = NAN;
        if (s.parts > 1) {
            float* to = slot_of<ROWS, D>(plan.states, s, s.part, kvh, nkv);
            const int row = M * wave + col;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < E; e += 4)
                    *reinterpret_cast<f4*>(to + row * D + M * i + G::key(e) + 4 * part) =
                        f4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
            if (part == 0) {
                to[ROWS * D + row] = m;
                to[ROWS * (D + 1) + row] = l;
            }
        } else {
            // (worked out again, not kept in registers over the loop)
            int row = w0 + col;
            asm("" : "+v"(row));
            const int tk = token_of(plan, row), hd = row - tk * plan.group;
            const float inv = s.kv - s.n + tk < 0 ? 0.0f : 1.0f / l;
            const int64_t at = (int64_t)(s.q0 + tk) * a.ld_out + (int64_t)(kvh * plan.group + hd) * D + 4 * part;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < E; e += 4)
                    store4(a, at + M * i + G::key(e), f4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]} * inv);
        }
    }
}

// ---- the join ------------------------------------------------------------------------------

constexpr int kJoinRows = 32, kJoinParts = 64;

// Joins kJoinRows rows of a tile of several parts: the parts' weights 2^(m - max m)
// through LDS, 64 parts at a time, and each output over the parts, by as many
// threads as there are for it.  In the parts' order, so with the same bits each time.
// Bound by the chain of loads for few parts (4 to 5 us, about 3 beside the attention's
// own end) and by the parts' bytes for many (34 MB for 512 tokens behind 15700, 10.6 us).
template <int D, int ROWS, int KEYS, class C>
__device__ __forceinline__ void join_part(const rf_paged_attention& a, const C& c, const Plan& plan, int item,
                                          float (*weight)[kJoinRows], f4* sums) {
    constexpr int JR = ROWS < kJoinRows ? ROWS : kJoinRows, SUB = ROWS / JR, LANES = 256 / JR;
    constexpr int PER = JR * (D / 4) / 256 > 1 ? JR * (D / 4) / 256 : 1;       // outputs a thread, of four
    const int nkv = c.num_kv_heads, tid = threadIdx.x;
    const int first = JR * (item % SUB), kvh = item / SUB % nkv;
    Share s;
    if (!find_share<ROWS, KEYS>(a, c, plan, item / SUB / nkv, true, s)) return;
    const int rows = s.n * plan.group, r0 = ROWS * s.tile;
    const int live = min(rows - r0 - first, JR);
    if (live <= 0) return;
    const int64_t next = (int64_t)s.tiles * nkv * (ROWS * (D + 2));
    const float* part0 = slot_of<ROWS, D>(plan.states, s, 0, kvh, nkv) + first * D;
    const float* m0 = part0 + (ROWS - first) * D + first;
    const int row = tid / LANES;                 // LANES lanes a row
    float mx = kNone, sum = 0.0f;
    if (row < live)
        for (int k = tid % LANES; k < s.parts; k += LANES) mx = fmaxf(mx, m0[k * next + row]);
    mx = xor_max<LANES / 2, 1>(mx);
    const int outs = live * (D / 4), groups = max(256 / outs, 1);
    const int g = groups == 1 ? 0 : tid / outs, i0 = groups == 1 ? tid : tid - g * outs;
    f4 acc[PER];
#pragma unroll
    for (int o = 0; o < PER; ++o) acc[o] = f4{0, 0, 0, 0};
    for (int k0 = 0; k0 < s.parts; k0 += kJoinParts) {
        const int n = min(s.parts - k0, kJoinParts);
        if (k0 > 0) __syncthreads();             // the last weights are read
        if (row < live)
            for (int k = tid % LANES; k < n; k += LANES) {
                const float f = __builtin_amdgcn_exp2f(m0[(k0 + k) * next + row] - mx);
                weight[k][row] = f;
                sum += m0[(k0 + k) * next + ROWS + row] * f;
            }
        __syncthreads();
        if (g < groups)
#pragma unroll
            for (int o = 0; o < PER; ++o) {
                const int i = i0 + 256 * o;
                if (i >= outs) continue;
#pragma unroll 4
                for (int k = g; k < n; k += groups)
                    acc[o] += *reinterpret_cast<const f4*>(part0 + (k0 + k) * next + 4 * i) * weight[k][i / (D / 4)];
            }
    }
    sum = xor_sum<LANES / 2, 1>(sum);
    __syncthreads();
    if (row < live && tid % LANES == 0)
        weight[0][row] = s.kv - s.n + token_of(plan, r0 + first + row) < 0 ? 0.0f : 1.0f / sum;
    sums[tid] = acc[0];
    __syncthreads();
    if (g > 0) return;
#pragma unroll
    for (int o = 0; o < PER; ++o) {
        const int i = i0 + 256 * o;
        if (i >= outs) continue;
        for (int k = 1; k < groups; ++k) acc[o] += sums[tid + k * outs];
        const int at = r0 + first + i / (D / 4), d = 4 * (i % (D / 4));
        const int tk = token_of(plan, at), hd = at - tk * plan.group;
        store4(a, (int64_t)(s.q0 + tk) * a.ld_out + (int64_t)(kvh * plan.group + hd) * D + d, acc[o] * weight[0][i / (D / 4)]);
    }
}

// Packed rows of a wide workgroup's tile, and the most wide parts that are aimed at: as many as fit the chip at once.
constexpr int kWideRows = 128;
template <int D>
constexpr int wide_parts() { return D == 256 ? 256 : 512; }

// Bytes of the narrow parts of a launch: twice as many as are aimed at; the wide ones' lie behind them.
template <int D>
constexpr size_t narrow_bytes() { return (size_t)2 * kNarrowParts * kNarrowRows * (D + 2) * sizeof(float); }
template <int D>
constexpr size_t wide_bytes() { return (size_t)2 * wide_parts<D>() * kWideRows * (D + 2) * sizeof(float); }

// ---- what the launchers refuse -------------------------------------------------------------

template <class C>
inline bool attention_ok(const rf_paged_attention& a, const C& c) {
    return a.num_seqs >= 0 && a.rows >= 0 && a.rows <= (1 << 23) && a.max_blocks >= 0 && a.num_heads > 0 &&
           a.num_heads <= 65535 && a.num_heads % c.num_kv_heads == 0 && a.num_heads / c.num_kv_heads <= 64 &&
           (int64_t)a.rows * a.num_heads <= (1 << 27) && a.window >= 0 && std::isfinite(a.scale) &&
           (int64_t)a.max_blocks * c.page_size <= (1 << 30);
}
template <class C>
inline bool attention_buffers_ok(const rf_paged_attention& a, const C& c) {
    const int64_t width = (int64_t)a.num_heads * c.head_dim;
    return a.q && a.out && a.block_tables && a.q_start && a.kv_lens && a.workspace && a.ld_q % 8 == 0 &&
           a.ld_out % 8 == 0 && a.ld_q >= width && a.ld_out >= width &&
           ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) |
             reinterpret_cast<uintptr_t>(a.workspace)) & 15u) == 0 &&
           a.workspace_bytes >= rf_paged_attention_workspace_bytes(a.num_heads, c.num_kv_heads, c.head_dim);
}

}  // namespace rf
