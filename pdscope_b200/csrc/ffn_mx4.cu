// Grouped SwiGLU experts on MXFP4 weights, on the block-scaled tensor cores:
//   y[p] = Wd (silu(Wg x) * (Wu x)),  x = x[tokens[p]], for every packed row p.
//
// The weights go to tcgen05.mma.kind::mxf8f6f4 as they are stored: E2M1 codes
// as the M operand (TMA unpacks them to one code per byte on the way to shared
// memory) and their E8M0 scales, one per 32 values of K, copied to TMEM.  No
// instruction is spent on dequantising, and HBM is read at 4.25 bits a weight.
//
// The activations keep BF16's precision in that 8-bit product as TWO E4M3
// pieces.  x and h are scaled by powers of two, one E8M0 scale per 32 values of K
// like the weights', that take a block's largest value into [128, 256):
//   hi = e4m3(v),  lo = e4m3(16 (v - hi)), read back through a scale of 1/16
// e4m3 keeps 4 significant bits, so |v - hi| <= 2^-4 |v|, which lo holds to
// 2^-9 |v|: an FP32 h is off by half of what rounding it to BF16 would cost, and a
// BF16 v (x) is represented exactly down to 2^-13 of its block's largest value;
// below that the error is at most 2^-14 (half of lo's smallest step), 2^-21 of the
// largest value.  A block of x that holds an infinity or NaN, and one of h where an
// infinity arises, is NaN throughout.
// W hi and W lo cost what one BF16 product would.
//
// Two launches of k_mx4_gemm, each on tiles of 256 weight rows (two accumulators
// over one token operand): 128 rows of gate and the same 128 of up with the
// SwiGLU, then 256 rows of down.  Tokens are the N operand, NT packed rows of
// one expert a tile.  Narrow tiles (NT = 16, 32) stack the two pieces along N (one
// pass over the weights in shared memory); wide ones (NT = 112, on pairs of CTAs)
// accumulate both into the same columns.
// Tiles go round robin over the CTAs, neighbours sharing a token tile in L2.  When
// there are fewer tiles than CTAs their K is cut up; a tile's parts are added in
// order by the warp that takes its last ticket (FP32, deterministic, nothing waits).
// Bound by HBM while an expert has few rows, by the power cap at prefill.  Device
// time of the three launches at H = 2048, I = 768, 128 experts, top-8, with the
// least the measured copy and BF16 rates allow: one token 16.2 us (3.1), 64 tokens
// 68-72 (48.5; 6.0-6.6 TB/s between the launches' starts and tails), 12,450 tokens
// 824-841 (578; 1.12-1.14 PFLOP/s).  The BF16 experts on the same packing, in turn
// with these: 23.2, 179 and 851 us; back to back for seconds, on the power cap, 12,450
// tokens take both 966 us (at 1455 MHz, these at 1327).
// Roles: warp 0 streams weights and scales, the last warp the token pieces, warp
// 1 issues the MMAs, the others are the epilogue (32 weight rows, = one scale
// block of h, and every second or fourth 8 token columns each).  Neither launch
// waits for another CTA (but for the other of its pair); the weight stream of a
// launch starts before the launch before it has finished.
#include <cuda.h>

#include "ffn_decode.cu"
#include "mxfp4.cu"
#include "tcgen05.cuh"

namespace pdx {

constexpr int kMx4MaxEpi = 16;                      // epilogue warps at most
constexpr int kMx4Chunk = 8;                        // token columns an epilogue warp takes at a time
constexpr int kMx4BK = 128;                         // K step: 4 MMAs of 32
constexpr uint32_t kMx4ABytes = 128 * kMx4BK;       // one weight tile, a byte per code
constexpr int kMx4TileBytes = 128 * kMx4BK / 2;     // its codes in memory
constexpr uint32_t kMx4SfBytes = 512;               // scales of 128 rows x 128 columns
constexpr int kMx4MaxActive = 1024;
constexpr uint32_t kMx4StageOut = 1024;             // 8 token columns x 64 weight rows on their way out
constexpr uint32_t kMx4TmemCols = 512;
constexpr uint32_t kMx4SfCol = 448;                 // 4 slots of weight and token scales, 4 columns a tile
constexpr int kMx4LoShift = 4;                      // lo pieces are held times 2^4
constexpr int kMx4SmemLimit = 227 * 1024;

// Scale byte b of a group from the bits of its largest magnitude, which 2^(127 - b)
// takes into [128, 256); 248 if the group holds an infinity or NaN; at least
// kMx4LoShift, so that the lo pieces' byte b - kMx4LoShift exists.
__device__ __forceinline__ uint32_t mx4_group_byte(uint32_t max_bits) {
    const uint32_t e = max_bits >> 23;
    return e > 7u + kMx4LoShift ? e - 7u : kMx4LoShift;
}
// 2^(127 - b), or NaN for a non-finite group: e4m3 has no infinity, and
// saturating would hide one.
__device__ __forceinline__ float mx4_inverse(uint32_t b) {
    return __uint_as_float(b < 248u ? (254u - b) << 23 : 0x7FC00000u);
}

// Two values -> their E4M3 pieces (a in the low byte).
__device__ __forceinline__ void e4m3_split2(float a, float b, uint16_t& hi, uint16_t& lo) {
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(b), "f"(a));
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(hi));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
    constexpr float up = 1 << kMx4LoShift;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"((b - f.y) * up), "f"((a - f.x) * up));
}

// Four BF16 values of x, scaled by inv: their E4M3 pieces by way of FP16, which holds
// a scaled BF16 exactly from 2^-17 up (below 2^-14 it is off by 2^-25 at most, where lo
// is off by 2^-14).
__device__ __forceinline__ void e4m3_split4(uint32_t a, uint32_t b, float inv, uint32_t& hi, uint32_t& lo) {
    uint16_t h[2], l[2];
    const uint32_t w[2] = {a, b};
    const __half2 up = __float2half2_rn(1 << kMx4LoShift);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2 v = __floats2half2_rn(__uint_as_float(w[i] << 16) * inv, __uint_as_float(w[i] & 0xFFFF0000u) * inv);
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(h[i]) : "r"(*reinterpret_cast<const uint32_t*>(&v)));
        uint32_t back;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(h[i]));
        const __half2 rest = __hmul2(__hsub2(v, *reinterpret_cast<const __half2*>(&back)), up);
        asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(l[i]) : "r"(*reinterpret_cast<const uint32_t*>(&rest)));
    }
    hi = h[0] | (static_cast<uint32_t>(h[1]) << 16);
    lo = l[0] | (static_cast<uint32_t>(l[1]) << 16);
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Where the split puts the scales of x: four bytes (of 128 columns) at `first + kb *
// step` for a row's hi piece, `lo` bytes further for its lo piece.
// Narrow token tiles: a 16-byte record per packed row and 128 columns, [kb][rows + 32]:
// any NT rows in a run are the scales of a token tile as tcgen05 wants them (hi in
// word 0, lo in word 1 at NT = 32, in a second array at NT = 16).  Wide ones: tiles of
// 512 bytes, [mx4_x_tile][kb][hi, lo].
struct Mx4Scales {
    uint8_t* bytes;
    int64_t step, lo;
};

// First scale tile of x of an expert whose packed rows start at seg0: experts of n
// rows have ceil(n / nt) tiles, which these starts keep apart whatever the list of
// active experts is; rows / nt + E in all.
__host__ __device__ constexpr int mx4_x_tile(int seg0, int e, int nt) { return seg0 / nt + e; }

// Token rows in packed order as E4M3 pieces: out [2][rows][Hp] (hi rows, then lo
// rows, zero past H) and a scale byte per 32 values.  A warp takes 512 UNROLL columns of
// a row, a lane 16 values at a time.  NT > 0: wide token tiles of NT rows, whose scales
// go by expert.  99,600 rows of 2048 take 110 us, 4.7 TB/s of DRAM traffic (the pieces
// are written once, x comes from L2 but for a third); 16 us of it are the scale bytes,
// which lie scattered over their tiles.  CTAs that collect the scales of 8, 16 or 32
// rows of a tile for whole sectors took 114, 103 and 101 us, and up to 8 us more than
// this at 1000 rows, where a warp then has several rows one after the other.  The
// kernel also clears the tickets of the two products that follow.
constexpr int kMx4SplitThreads = 128;
template <int UNROLL, int NT>
__global__ void __launch_bounds__(kMx4SplitThreads, UNROLL == 1 ? 12 : (UNROLL == 2 ? 10 : 7))
    k_mx4_split(const uint16_t* __restrict__ x, const int32_t* __restrict__ tokens, int T, int rows, int H, int Hp,
                uint8_t* __restrict__ out, Mx4Scales scales, const int32_t* __restrict__ offsets, int E,
                unsigned int* __restrict__ zero_ptr, int zero_words) {
    griddep_wait();
    griddep_launch();
    __shared__ int s_off[NT ? kMx4MaxActive + 1 : 1];
    for (int i = static_cast<int>(blockIdx.x * blockDim.x + threadIdx.x); i < zero_words;
         i += static_cast<int>(gridDim.x * blockDim.x))
        zero_ptr[i] = 0u;
    if (NT) {
        for (int i = static_cast<int>(threadIdx.x); i <= kMx4MaxActive; i += kMx4SplitThreads)
            s_off[i] = i <= E ? __ldg(offsets + i) : rows;
        __syncthreads();
    }
    constexpr int kWarps = kMx4SplitThreads / 32;
    const int lane = static_cast<int>(lane_id()), sub = lane & 7;
    const int chunks = H / 16, chunks_p = Hp / 16, per_row = (chunks_p + 32 * UNROLL - 1) / (32 * UNROLL);
    const int units = rows * per_row;
    const uint32_t odd = sub & 1, minus = odd ? kMx4LoShift : 0;       // even lanes store scales of hi, odd ones of lo
    for (int u = static_cast<int>(blockIdx.x * kWarps + threadIdx.x / 32); u < units;
         u += static_cast<int>(gridDim.x) * kWarps) {
        const int p = per_row == 1 ? u : u / per_row, c0 = (u - p * per_row) * (32 * UNROLL) + lane;
        int t = tokens ? __ldg(tokens + p) : p;
        if (t < 0 || t >= T) {
            raise_error(PDX_DEVERR_BAD_EXPERT);
            t = 0;
        }
        const uint4* src = reinterpret_cast<const uint4*>(x + static_cast<int64_t>(t) * H) + 2 * c0;
        uint4 v[UNROLL][2];
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            v[j][0] = c0 + 32 * j < chunks ? __ldg(src + 64 * j) : make_uint4(0, 0, 0, 0);
            v[j][1] = c0 + 32 * j < chunks ? __ldg(src + 64 * j + 1) : make_uint4(0, 0, 0, 0);
        }
        int64_t first = 16 * static_cast<int64_t>(p);
        bool scaled = true;
        if (NT) {
            // the last expert that starts at p or before, in two steps of 32
            static_assert(kMx4MaxActive == 32 * 32, "two steps");
            int e = 32 * (__popc(__ballot_sync(0xffffffffu, s_off[32 * lane] <= p)) - 1);
            e += __popc(__ballot_sync(0xffffffffu, s_off[max(e, 0) + lane] <= p)) - 1;
            e = min(max(e, 0), E - 1);
            const int seg0 = s_off[e], r = p - seg0;
            // a row of no expert is in no tile and has no scales
            scaled = seg0 >= 0 && r >= 0 && p < s_off[e + 1];
            first = (mx4_x_tile(seg0, e, NT) + r / NT) * (chunks_p * int64_t(128)) + (r % NT % 32) * 16 + r % NT / 32 * 4;
        }
        uint8_t* to = scales.bytes + first + (c0 >> 3) * scales.step + (odd ? scales.lo : 0) + (sub >> 1);
        uint4* hi_row = reinterpret_cast<uint4*>(out + static_cast<int64_t>(p) * Hp) + c0;
        uint4* lo_row = reinterpret_cast<uint4*>(out + (static_cast<int64_t>(rows) + p) * Hp) + c0;
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            const uint32_t w[8] = {v[j][0].x, v[j][0].y, v[j][0].z, v[j][0].w,
                                   v[j][1].x, v[j][1].y, v[j][1].z, v[j][1].w};
            uint32_t two = w[0] & 0x7FFF7FFFu;                 // the largest magnitudes of the even and of the odd values
#pragma unroll
            for (int i = 1; i < 8; ++i) two = max_u16x2(two, w[i] & 0x7FFF7FFFu);
            two = max_u16x2(two, __shfl_xor_sync(0xffffffffu, two, 1));   // two lanes hold a block of 32
            const uint32_t byte = mx4_group_byte(max(two << 16, two & 0xFFFF0000u));
            const float inv = mx4_inverse(byte);
            uint32_t h[4], l[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e4m3_split4(w[2 * i], w[2 * i + 1], inv, h[i], l[i]);
            if (c0 + 32 * j < chunks_p) {                      // eight lanes, 128 columns, alike
                __stcs(hi_row + 32 * j, make_uint4(h[0], h[1], h[2], h[3]));   // streaming: x stays in L2
                __stcs(lo_row + 32 * j, make_uint4(l[0], l[1], l[2], l[3]));
                if (scaled) to[4 * j * scales.step] = static_cast<uint8_t>(byte - minus);   // kMx4LoShift at least
            }
        }
    }
}

struct Mx4Args {
    const int32_t* offsets;         // [E+1]
    const int32_t* active;          // [E+1] active count, then the active expert ids
    const int32_t* slot_of_expert;  // NULL = identity
    int64_t num_slots;
    const uint8_t* scales;          // weight scales of slot 0
    int64_t scale_stride;           // bytes between slots
    int64_t tiles_per_slot;         // weight tiles between slots
    int tile0, tile1;               // first weight tile of gate and up, or of down (tile0)
    int K, M;                       // multiples of 128: reduction length, weight rows
    int rows;
    const uint8_t* xs;              // x scales of narrow token tiles (Mx4Scales), x_pad records per 128 columns (SWIGLU)
    int x_pad;
    uint8_t* sf;                    // h scales: [token tile][Ip / 128][kSfTiles] tiles of 512 bytes (out of SWIGLU, else in)
    uint8_t* h;                     // [2][rows][M] pieces (SWIGLU)
    uint16_t* y;                    // [rows, ldy] (down)
    int ldy;                        // H
    int stages, table;              // ring stages, entries of the expert tables: E
    int max_tiles;                  // token tiles that sf has room for
    float* partials;                // [gridDim.x][2 NT][128]
    unsigned int* tickets;          // [CTAs * epilogue warps], zero on entry
};

// Four words of four bytes, transposed: byte i of the words -> out[i].
__device__ __forceinline__ void turn_bytes(const uint4& w, uint32_t (&out)[4]) {
    const uint32_t a = __byte_perm(w.x, w.y, 0x5140), b = __byte_perm(w.z, w.w, 0x5140);
    const uint32_t c = __byte_perm(w.x, w.y, 0x7362), d = __byte_perm(w.z, w.w, 0x7362);
    out[0] = __byte_perm(a, b, 0x5410);
    out[1] = __byte_perm(a, b, 0x7632);
    out[2] = __byte_perm(c, d, 0x5410);
    out[3] = __byte_perm(c, d, 0x7632);
}

// One more of the parts of a tile is stored: the parts written before it (by the
// lanes of this warp, behind __syncwarp) are visible to whoever sees the count.
__device__ __forceinline__ unsigned int ticket_acq_rel(unsigned int* p) {
    unsigned int v;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(v) : "l"(p) : "memory");
    return v;
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

__device__ __forceinline__ uint64_t mx4_sf_desc(uint32_t smem_addr) {  // 32 x 16 bytes, 8-row groups 128 bytes apart
    return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(128 >> 4) << 32) |
           (static_cast<uint64_t>(1) << 46);
}

// A = E2M1 (5), B = E4M3 (0), E8M0 scales; the scale byte of the K step is or'ed in.
__host__ __device__ constexpr uint32_t mx4_idesc(int m, int n) {
    return (5u << 7) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(m >> 7) << 27);
}

template <bool PAIR>
__device__ __forceinline__ void umma_mx4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::
                "r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::
                "r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate));
}

// 512 bytes of scales from shared memory to four TMEM columns (PAIR: in both
// CTAs, each from its own shared memory).
template <bool PAIR>
__device__ __forceinline__ void tmem_cp_sf(uint32_t taddr, uint64_t desc) {
    if (PAIR)
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
            smem_u32(smem_dst)),
        "l"(src), "r"(bytes), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const void* tmap, uint32_t bar_cluster_addr, int32_t x,
                                                 int32_t y, int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
        "%5}], [%2];" ::"r"(smem_u32(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const void* tmap, uint64_t* bar, int32_t x, int32_t y,
                                            int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(smem_u32(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}

template <int NT>
struct Mx4Shape {
    static constexpr bool kPair = NT > 32;                          // two CTAs share a tile
    static constexpr bool kStack = !kPair;                          // pieces side by side along N
    static constexpr int kN = kStack ? 2 * NT : NT;                 // N of one MMA
    static constexpr int kAcc = 2 * kN;                             // accumulator columns of a tile
    static constexpr int kCols = 2 * NT;                            // FP32 columns of a partial tile
    static constexpr int kBRows = kPair ? NT / 2 : NT;               // token rows a CTA stages
    static constexpr uint32_t kA = 2 * kMx4ABytes;
    static constexpr uint32_t kATx = kA / 2;                        // the copy counts the packed bytes it reads
    static constexpr uint32_t kB = 2 * kBRows * kMx4BK;
    static constexpr uint32_t kStage = kA + kB;                     // multiple of 1024
    static constexpr int kSfTiles = kStack ? 1 : 2;                 // token scales: stacked, or hi | lo
    static constexpr uint32_t kSf = (2 + kSfTiles) * kMx4SfBytes;   // both weight halves | tokens
    // Eight columns take one of eight epilogue warps 1000 (down) to 2000 cycles
    // (SwiGLU), mostly latency.  Wide tiles have 14 such pieces to 6 K steps of MMAs
    // (5600 cycles at NT = 112, I = 768), so they take 16 warps (prefill 884 -> 846 us);
    // narrow ones keep the shared memory for the ring.
    static constexpr int kEpi = kPair ? 16 : 8;
    static constexpr int kThreads = 32 * (kEpi + 3);
    static constexpr uint32_t kFixed = 1024 + 512 + kEpi * kMx4StageOut;   // alignment, barriers, staging
    static constexpr uint32_t kEntry = kPair ? 20 : 16;                    // an expert's entry in the tables
    // Ring stages beside tables of `entries` experts, and the shared memory of both.
    static constexpr int stages(int entries) {
        return static_cast<int>((kMx4SmemLimit - kFixed - kEntry * entries) / (kStage + kSf));
    }
    static constexpr size_t smem(int entries) { return kFixed + kEntry * entries + stages(entries) * (kStage + kSf); }
    static constexpr int kMaxStages = stages(1);
    static_assert(NT % 16 == 0 && kBRows % 8 == 0 && stages(kMx4MaxActive) >= 3 && 2 * kMaxStages + 5 <= 56 &&
                      2 * kAcc <= static_cast<int>(kMx4SfCol),
                  "token tile");
};

// NT > 32: a cluster of two CTAs shares a tile of 512 weight rows (tcgen05
// cta_group::2): each CTA stages its own 256 weight rows and half of the token
// rows, rank 0 issues the MMAs for both, each CTA's TMEM holds the sums of its own
// weight rows.  Token bytes from L2 and their shared memory are halved, which
// leaves room for a fourth stage at NT = 112.  Rank 0's full barriers count the
// bytes of both CTAs; rank 0 commits to the empty and TMEM barriers of both.
template <int NT, bool SWIGLU>
__global__ void __launch_bounds__(Mx4Shape<NT>::kThreads, 1)
    k_mx4_gemm(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
               const __grid_constant__ CUtensorMap tm_ws, const __grid_constant__ CUtensorMap tm_xs, Mx4Args args) {
    using S = Mx4Shape<NT>;
    constexpr bool PAIR = S::kPair;
    constexpr int kCtas = PAIR ? 2 : 1;
    // K steps of a part of a tile, at least.  Joining wide parts costs more (T = 200,
    // two experts, H = 4096, I = 1536: parts of 4 steps 47 us, 8 39, uncut 39; one
    // token, two experts of 16, H = 2048, I = 768: parts of 4 steps 12.8, 8 14.0).
    constexpr int kMinPart = PAIR ? 16 : 4;
    constexpr int kJoin = PAIR ? 1 : 4;                      // parts in flight when a tile is joined
    constexpr int kColStep = S::kEpi / 4 * kMx4Chunk;        // columns between an epilogue warp's chunks
    extern __shared__ __align__(1024) unsigned char smem_mx4[];
    unsigned char* smem = smem_mx4 + ((1024u - (smem_u32(smem_mx4) & 1023u)) & 1023u);
    const int stages = args.stages;
    unsigned char* s_sf = smem + stages * S::kStage;                 // stages x kSf
    unsigned char* s_bar = s_sf + stages * S::kSf;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(s_bar);
    uint64_t* empty_bar = full_bar + stages;
    uint64_t* tmem_full = empty_bar + stages;
    uint64_t* tmem_empty = tmem_full + 2;
    uint64_t* drain_bar = tmem_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* s_misc = reinterpret_cast<int*>(tmem_slot + 2);
    unsigned char* s_out = s_bar + 512;                              // an epilogue warp's staging: kMx4StageOut
    int* prefix = reinterpret_cast<int*>(s_out + S::kEpi * kMx4StageOut);   // token tiles before an active expert
    int* t_seg0 = prefix + args.table;
    int* t_rows = t_seg0 + args.table;
    int* t_slot = t_rows + args.table;
    int* t_xs = t_slot + args.table;                                 // PAIR: first scale tile of x

    const int warp = static_cast<int>(threadIdx.x >> 5);
    const uint32_t lane = lane_id();
    const int m_blocks = args.M / 128, nkb = args.K / kMx4BK;
    constexpr int kTileBlocks = (SWIGLU ? 1 : 2) * kCtas;    // 128-row blocks of M a tile covers
    const int m_tiles = (m_blocks + kTileBlocks - 1) / kTileBlocks;
    const int rank = PAIR ? static_cast<int>(cluster_ctarank()) : 0;
    const uint32_t peer_abort =
        PAIR ? mapa_shared(smem_u32(const_cast<int*>(abort_flag)), static_cast<uint32_t>(rank ^ 1)) : 0u;
    // Bounded wait; running out releases the other roles, and the other CTA.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_wait(bar, parity, abort_flag)) return true;
        if (PAIR) st_shared_remote_u32(peer_abort, 1u);
        return false;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tmem_full[b], 1);
            mbar_init(&tmem_empty[b], kCtas * S::kEpi);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_x);
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile(
                "tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                "r"(kMx4TmemCols)
                : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile(
                "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                "r"(kMx4TmemCols)
                : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    // The routing tables are older than the launch before this one, which has
    // passed its own wait by the time this one starts; only that launch's
    // output (the token pieces) has to be waited for, by the warps that read it.
    // The list may name experts without rows, but none outside [0, E) and no more
    // than E; an expert's rows lie in [0, rows).  What breaks that has no rows here.
    const int listed = __ldcg(args.active), n_active = max(0, min(listed, args.table));
    if (listed != n_active && threadIdx.x == 0) raise_error(PDX_DEVERR_BAD_EXPERT);
    for (int i = static_cast<int>(threadIdx.x); i < n_active; i += S::kThreads) {
        int e = __ldcg(args.active + 1 + i);
        const bool known = e >= 0 && e < args.table;
        if (!known) e = 0;
        int seg0 = __ldcg(args.offsets + e), end = __ldcg(args.offsets + e + 1);
        if (!known || seg0 < 0 || end < seg0 || end > args.rows) {
            raise_error(PDX_DEVERR_BAD_EXPERT);
            seg0 = end = 0;
        }
        int64_t slot = args.slot_of_expert ? __ldcg(args.slot_of_expert + e) : e;
        if (slot < 0 || slot >= args.num_slots) {
            raise_error(PDX_DEVERR_BAD_SLOT);
            slot = 0;
        }
        t_seg0[i] = seg0;
        t_rows[i] = end - seg0;
        t_slot[i] = static_cast<int>(slot);
        if (PAIR) t_xs[i] = mx4_x_tile(seg0, e, NT);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 2) {
        const int total = warp_tile_prefix(n_active, prefix, [&](int a) { return (t_rows[a] + NT - 1) / NT; });
        if (lane == 0) {
            if (total > args.max_tiles) raise_error(PDX_DEVERR_BAD_EXPERT);   // an expert listed again and again
            s_misc[0] = min(total, args.max_tiles) * m_tiles;
        }
    }
    __syncwarp();
    if (PAIR)
        cluster_sync_all();   // both CTAs' barriers are initialised before any remote arrival
    else
        __syncthreads();
    const uint32_t full0 = PAIR ? mapa_shared(smem_u32(full_bar), 0) : 0u;          // rank 0's barriers
    const uint32_t tmem_empty0 = PAIR ? mapa_shared(smem_u32(tmem_empty), 0) : 0u;
    const uint32_t tmem_base = *tmem_slot;
    // CTA (or pair) c of G takes the tiles c, c + G, ...  When there are fewer tiles
    // than CTAs (a few tokens), K is cut into `parts` equal parts of at least
    // kMinPart steps and CTA c takes part c % parts of tile c / parts: one token at
    // H = 2048, I = 768, 8 experts has 48 gate/up tiles of 16 steps (3 parts) and 64
    // down tiles of 6 (1 part).  Cutting up the last, partial wave of many tiles the
    // same way costs more in joining than it evens out (T = 2048: 225 us against 215,
    // T = 1024 at H = 1024, I = 512, 32 experts: 42 against 35).
    const int grid = static_cast<int>(gridDim.x) / kCtas, cta = static_cast<int>(blockIdx.x) / kCtas;
    const int tiles = s_misc[0];
    const int parts = max(1, min(grid / max(tiles, 1), nkb / kMinPart));

    struct Tile {
        int unit;                                  // tile * parts + part
        int index, token, a, mt, nb, kb0, kb1;     // tile, its token tile, expert, weight tile, tile of the expert, steps
    };
    auto next = [&](Tile& t) {
        t.unit += grid;
        if (t.unit >= tiles * parts) return false;
        t.index = t.unit / parts;
        const int part = t.unit - t.index * parts;
        t.kb0 = part * nkb / parts;
        t.kb1 = (part + 1) * nkb / parts;
        t.token = t.index / m_tiles;
        t.mt = t.index - t.token * m_tiles;
        t.a = find_expert(prefix, n_active, t.token);
        t.nb = t.token - prefix[t.a];
        return true;
    };
    auto begin = [&]() {
        Tile t;
        t.unit = cta - grid;
        return t;
    };

    if (warp == 0) {
        // ---------------- weight producer ----------------
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (Tile t = begin(); ok && next(t);) {
                const int64_t slot = t_slot[t.a];
                // weight tiles of both halves; blocks past the last are loaded again and not used
                const int blk = t.mt * kTileBlocks + rank * (SWIGLU ? 1 : 2), end = m_blocks - 1;
                const int b0 = args.tile0 + min(blk, end) * nkb;
                const int b1 = SWIGLU ? args.tile1 + min(blk, end) * nkb : args.tile0 + min(blk + 1, end) * nkb;
                const int64_t tile0 = slot * args.tiles_per_slot;
                const uint8_t* sf = args.scales + slot * args.scale_stride;
                const int sf_row = static_cast<int>(slot * (args.scale_stride / kMx4SfBytes));
                for (int kb = t.kb0; kb < t.kb1; ++kb) {
                    if (!wait(&empty_bar[stage], phase ^ 1u)) { ok = false; break; }
                    unsigned char* sa = smem + stage * S::kStage;
                    unsigned char* ss = s_sf + stage * S::kSf;
                    const int y0 = static_cast<int>(tile0 + b0 + kb) * 128, y1 = static_cast<int>(tile0 + b1 + kb) * 128;
                    if (rank == 0)
                        mbar_arrive_expect_tx(&full_bar[stage],
                                              kCtas * (S::kATx + S::kB + (2 + S::kSfTiles) * kMx4SfBytes));
                    if (PAIR) {
                        const uint32_t fb = full0 + static_cast<uint32_t>(stage) * 8u;
                        tma_load_2d_pair(sa, &tm_w, fb, 0, y0);
                        tma_load_2d_pair(sa + kMx4ABytes, &tm_w, fb, 0, y1);
                        tma_load_2d_pair(ss, &tm_ws, fb, 0, sf_row + b0 + kb);
                        tma_load_2d_pair(ss + kMx4SfBytes, &tm_ws, fb, 0, sf_row + b1 + kb);
                    } else {
                        tma_load_2d(sa, &tm_w, &full_bar[stage], 0, y0);
                        tma_load_2d(sa + kMx4ABytes, &tm_w, &full_bar[stage], 0, y1);
                        bulk_load(ss, sf + static_cast<int64_t>(b0 + kb) * kMx4SfBytes, kMx4SfBytes, &full_bar[stage]);
                        bulk_load(ss + kMx4SfBytes, sf + static_cast<int64_t>(b1 + kb) * kMx4SfBytes, kMx4SfBytes,
                                  &full_bar[stage]);
                    }
                    if (++stage == stages) { stage = 0; phase ^= 1u; }
                }
            }
            // PAIR: every stage's last release (a commit of rank 0) has landed before
            // this CTA's shared memory can go away
            for (int i = 0; PAIR && i < stages && ok; ++i) {
                ok = wait(&empty_bar[stage], phase ^ 1u);
                if (++stage == stages) { stage = 0; phase ^= 1u; }
            }
        }
        __syncwarp();
    } else if (warp == 2 + S::kEpi) {
        // ---------------- token producer ----------------
        griddep_wait();
        griddep_launch();
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (Tile t = begin(); ok && next(t);) {
                const int row = t_seg0[t.a] + t.nb * NT + rank * S::kBRows;
                const int64_t tt = PAIR && SWIGLU ? t_xs[t.a] + t.nb : t.token;   // scale tiles of x, of h
                for (int kb = t.kb0; kb < t.kb1; ++kb) {
                    if (!wait(&empty_bar[stage], phase ^ 1u)) { ok = false; break; }
                    if (PAIR) {
                        const uint32_t fb = full0 + static_cast<uint32_t>(stage) * 8u;
                        tma_load_3d_pair(smem + stage * S::kStage + S::kA, &tm_x, fb, kb * kMx4BK, row, 0);
                        for (int i = 0; i < S::kSfTiles; ++i)
                            tma_load_2d_pair(s_sf + stage * S::kSf + (2 + i) * kMx4SfBytes, &tm_xs, fb, 0,
                                             static_cast<int>(tt * nkb + kb) * S::kSfTiles + i);
                        if (++stage == stages) { stage = 0; phase ^= 1u; }
                        continue;
                    }
                    tma_load_3d(smem + stage * S::kStage + S::kA, &tm_x, &full_bar[stage], kb * kMx4BK, row, 0);
                    unsigned char* ss = s_sf + stage * S::kSf + 2 * kMx4SfBytes;
                    if (SWIGLU) {
                        const int64_t record = static_cast<int64_t>(kb) * args.x_pad + row;
                        for (int i = 0; i < 32 / NT; ++i)                        // 32 records; NT = 16: of hi, then of lo
                            bulk_load(ss + i * (NT * 16), args.xs + (static_cast<int64_t>(i) * nkb * args.x_pad + record) * 16,
                                      NT * 16, &full_bar[stage]);
                    } else {
                        bulk_load(ss, args.sf + (tt * nkb + kb) * kMx4SfBytes, kMx4SfBytes, &full_bar[stage]);
                    }
                    if (++stage == stages) { stage = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {
        // ---------------- MMA issuer (of the pair: rank 0) ----------------
        constexpr uint32_t idesc = mx4_idesc(128 * kCtas, S::kN);
        constexpr uint32_t kSlot = 8 + 4 * S::kSfTiles;   // scale columns of a K step
        auto commit = [&](uint64_t* bar) {   // to this barrier of every CTA of the tile
            if (PAIR) {
                umma_commit_pair(smem_u32(bar));
                umma_commit_pair(mapa_shared(smem_u32(bar), 1));
            } else {
                umma_commit(bar);
            }
        };
        int stage = 0, lt = 0, step = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (Tile t = begin(); ok && next(t); ++lt) {
            const int b = lt & 1;
            const uint32_t acc_phase = static_cast<uint32_t>(lt >> 1) & 1u;
            if (!wait(&tmem_empty[b], acc_phase ^ 1u)) { ok = false; break; }
            tc_fence_after();
            const uint32_t d = tmem_base + static_cast<uint32_t>(b * S::kAcc);
            for (int kb = t.kb0; kb < t.kb1; ++kb, ++step) {
                if (!wait(&full_bar[stage], phase)) { ok = false; break; }
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t sa = smem_u32(smem + stage * S::kStage);
                    const uint32_t ss = smem_u32(s_sf + stage * S::kSf);
                    const uint32_t sf = tmem_base + kMx4SfCol + static_cast<uint32_t>(step & 3) * kSlot;
                    tmem_cp_sf<PAIR>(sf, mx4_sf_desc(ss));
                    tmem_cp_sf<PAIR>(sf + 4, mx4_sf_desc(ss + kMx4SfBytes));
                    for (int i = 0; i < S::kSfTiles; ++i)
                        tmem_cp_sf<PAIR>(sf + 8 + 4 * i, mx4_sf_desc(ss + (2 + i) * kMx4SfBytes));
                    const uint32_t sfb = sf + 8, sfb_lo = sfb + 4;
                    const uint64_t a0 = sw128_desc(sa), a1 = sw128_desc(sa + kMx4ABytes);
                    const uint64_t hi = sw128_desc(sa + S::kA), lo = sw128_desc(sa + S::kA + S::kBRows * kMx4BK);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint32_t acc = (kb > t.kb0 || kk > 0) ? 1u : 0u;
                        const uint32_t id = idesc | (static_cast<uint32_t>(kk) << 29) | (static_cast<uint32_t>(kk) << 4);
                        umma_mx4<PAIR>(d, a0 + 2u * kk, hi + 2u * kk, id, sf, sfb, acc);
                        if (!S::kStack) umma_mx4<PAIR>(d, a0 + 2u * kk, lo + 2u * kk, id, sf, sfb_lo, 1u);
                        umma_mx4<PAIR>(d + S::kN, a1 + 2u * kk, hi + 2u * kk, id, sf + 4, sfb, acc);
                        if (!S::kStack) umma_mx4<PAIR>(d + S::kN, a1 + 2u * kk, lo + 2u * kk, id, sf + 4, sfb_lo, 1u);
                    }
                    commit(&empty_bar[stage]);
                }
                __syncwarp();
                if (++stage == stages) { stage = 0; phase ^= 1u; }
            }
            if (!ok) break;
            if (elect_one()) commit(&tmem_full[b]);
            __syncwarp();
        }
    } else if (warp >= 2) {
        // ---------------- epilogue (S::kEpi warps from 2) ----------------
        griddep_wait();
        const int q = warp & 3;                                  // TMEM lane quadrant
        const int col0 = ((warp - 2) >> 2) * kMx4Chunk;          // first columns of this warp
        const int i_row = q * 32 + static_cast<int>(lane);
        // Staged words are read 32 bytes a lane; in every second group of 32 words the
        // 16-byte halves change places, so eight lanes read eight different bank groups.
        const uint32_t turn = lane >> 2 & 1u;
        uint32_t* out = reinterpret_cast<uint32_t*>(s_out + (warp - 2) * kMx4StageOut);
        // Token columns [c0, c0 + n), n <= 8, of a tile: the sums g of the first, u of the second 128 weight rows.
        auto finish = [&](const Tile& t, int c0, int n, float (&g)[kMx4Chunk], float (&u)[kMx4Chunk]) {
            const int64_t p0 = static_cast<int64_t>(t_seg0[t.a]) + t.nb * NT + c0;
            const int part = t.mt * kCtas + rank;                // of the tiles of 256 weight rows
            if (SWIGLU) {
                if (part >= m_blocks) return;
                uint32_t byte = 0;                               // lane j: scale byte of column j
                uint32_t top[kMx4Chunk];
#pragma unroll
                for (int j = 0; j < kMx4Chunk; ++j) {
                    g[j] = __fdividef(g[j], 1.0f + __expf(-g[j])) * u[j];
                    // the 32 lanes are one scale block of h
                    top[j] = __reduce_max_sync(0xffffffffu, __float_as_uint(g[j]) & 0x7FFFFFFFu);
                }
#pragma unroll
                for (int j = 0; j < kMx4Chunk; ++j) {
                    const uint32_t by = mx4_group_byte(top[j]);
                    g[j] *= mx4_inverse(by);
                    if (static_cast<int>(lane) == j) byte = by;
                }
                // One word per weight row and 4 columns, [4 columns][piece][32 rows]; then half the
                // lanes take 8 rows of 4 columns of a piece, turn them and store 8 bytes a column.
#pragma unroll
                for (int j = 0; j < kMx4Chunk; j += 4) {
                    uint16_t h0, h1, l0, l1;
                    e4m3_split2(g[j], g[j + 1], h0, l0);
                    e4m3_split2(g[j + 2], g[j + 3], h1, l1);
                    out[16 * j + lane] = h0 | (static_cast<uint32_t>(h1) << 16);
                    out[16 * j + 32 + (lane ^ 4)] = l0 | (static_cast<uint32_t>(l1) << 16);   // see turn
                }
                __syncwarp();
                if (lane < 16) {
                    const int j = (static_cast<int>(lane) >> 3) * 4, piece = (static_cast<int>(lane) >> 2) & 1;
                    const uint4 w0 = reinterpret_cast<const uint4*>(out)[2 * lane ^ turn];
                    const uint4 w1 = reinterpret_cast<const uint4*>(out)[(2 * lane + 1) ^ turn];
                    uint32_t a[4], b[4];
                    turn_bytes(w0, a);
                    turn_bytes(w1, b);
                    uint8_t* at = args.h + (piece * static_cast<int64_t>(args.rows) + p0 + j) * args.M + part * 128 +
                                  q * 32 + (lane & 3) * 8;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (j + i < n) *reinterpret_cast<uint2*>(at) = make_uint2(a[i], b[i]);
                        at += args.M;
                    }
                }
                __syncwarp();
                if (lane < kMx4Chunk) {
                    const int r = c0 + static_cast<int>(lane);   // row of the token tile
                    uint8_t* sf =
                        args.sf + (static_cast<int64_t>(t.token) * m_blocks + part) * (S::kSfTiles * kMx4SfBytes) + q;
                    const int hi_at = (r & 31) * 16 + (r >> 5) * 4;
                    const int lo_at = S::kStack ? ((r + NT) & 31) * 16 + ((r + NT) >> 5) * 4 : hi_at + kMx4SfBytes;
                    sf[hi_at] = static_cast<uint8_t>(byte);
                    sf[lo_at] = static_cast<uint8_t>(byte - kMx4LoShift);
                }
            } else {
                // One word per weight row and 2 columns, [half][2 columns][32 rows]; then every
                // lane takes 8 rows of 2 columns, turns them and stores 16 bytes a column.
                const int col = part * 256 + q * 32;             // H is a multiple of 32: all lanes in or out
#pragma unroll
                for (int j = 0; j < kMx4Chunk; j += 2) {
                    const uint32_t at = 16 * j + (lane ^ (j & 2 ? 4u : 0u));                  // see turn
                    out[at] = f2bits(g[j]) | (static_cast<uint32_t>(f2bits(g[j + 1])) << 16);
                    out[128 + at] = f2bits(u[j]) | (static_cast<uint32_t>(f2bits(u[j + 1])) << 16);
                }
                __syncwarp();
                const int c8 = col + (static_cast<int>(lane) >> 4) * 128, j = (static_cast<int>(lane) >> 2 & 3) * 2;
                const uint4 w0 = reinterpret_cast<const uint4*>(out)[2 * lane ^ turn];
                const uint4 w1 = reinterpret_cast<const uint4*>(out)[(2 * lane + 1) ^ turn];
                uint16_t* at = args.y + (p0 + j) * args.ldy + c8 + (lane & 3) * 8;
                if (j < n && c8 < args.ldy)
                    *reinterpret_cast<uint4*>(at) =
                        make_uint4(__byte_perm(w0.x, w0.y, 0x5410), __byte_perm(w0.z, w0.w, 0x5410),
                                   __byte_perm(w1.x, w1.y, 0x5410), __byte_perm(w1.z, w1.w, 0x5410));
                if (j + 1 < n && c8 < args.ldy)
                    *reinterpret_cast<uint4*>(at + args.ldy) =
                        make_uint4(__byte_perm(w0.x, w0.y, 0x7632), __byte_perm(w0.z, w0.w, 0x7632),
                                   __byte_perm(w1.x, w1.y, 0x7632), __byte_perm(w1.z, w1.w, 0x7632));
                __syncwarp();
            }
        };
        auto release = [&](int b) {                              // this warp has read accumulator b
            tc_fence_before();
            __syncwarp();
            if (lane != 0) return;
            if (PAIR)
                mbar_arrive_remote(tmem_empty0 + static_cast<uint32_t>(b) * 8u);
            else
                mbar_arrive(&tmem_empty[b]);
        };
        int lt = 0;
        for (Tile t = begin(); next(t); ++lt) {
            const int b = lt & 1;
            const uint32_t acc_phase = static_cast<uint32_t>(lt >> 1) & 1u;
            const int ne = min(NT, t_rows[t.a] - t.nb * NT);     // rows of the tile
            if (!wait(&tmem_full[b], acc_phase)) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(b * S::kAcc);
            // a part's sums; with parts > 1 a CTA has one unit
            float* mine = args.partials + static_cast<int64_t>(blockIdx.x) * S::kCols * 128 + i_row;
            for (int c = col0; c < ne; c += kColStep) {
                const int n = min(kMx4Chunk, ne - c);
                uint32_t r[4][kMx4Chunk];
                tmem_ld8(taddr + c, r[0]);
                tmem_ld8(taddr + S::kN + c, r[1]);
                if (S::kStack) {
                    tmem_ld8(taddr + NT + c, r[2]);
                    tmem_ld8(taddr + S::kN + NT + c, r[3]);
                }
                tmem_wait_ld();
                if (c + kColStep >= ne) release(b);         // this warp's last columns are read
                float g[kMx4Chunk], u[kMx4Chunk];
#pragma unroll
                for (int j = 0; j < kMx4Chunk; ++j) {
                    g[j] = __uint_as_float(r[0][j]) + (S::kStack ? __uint_as_float(r[2][j]) : 0.f);
                    u[j] = __uint_as_float(r[1][j]) + (S::kStack ? __uint_as_float(r[3][j]) : 0.f);
                }
                if (parts == 1) {
                    finish(t, c, n, g, u);
                } else {
#pragma unroll
                    for (int j = 0; j < kMx4Chunk; ++j)
                        if (j < n) {
                            mine[(c + j) * 128] = g[j];
                            mine[(NT + c + j) * 128] = u[j];
                        }
                }
            }
            if (col0 >= ne) release(b);
            if (parts == 1) continue;
            // the warp that takes a tile's last ticket adds the parts, in their order
            __syncwarp();
            unsigned int prev = 0;
            if (lane == 0) prev = ticket_acq_rel(&args.tickets[(t.index * kCtas + rank) * S::kEpi + warp - 2]);
            prev = __shfl_sync(0xffffffffu, prev, 0);
            if (prev != static_cast<unsigned int>(parts - 1)) continue;
            __syncwarp();   // lane 0 acquired the other CTAs' parts; this orders it before the reads of all lanes
            for (int col = col0; col < ne; col += kColStep) {
                const int n = min(kMx4Chunk, ne - col);
                float g[kMx4Chunk], u[kMx4Chunk];
#pragma unroll
                for (int j = 0; j < kMx4Chunk; ++j) g[j] = u[j] = 0.f;
#pragma unroll kJoin
                for (int i = 0; i < parts; ++i) {
                    const float* p = args.partials +
                                     static_cast<int64_t>((t.index * parts + i) * kCtas + rank) * S::kCols * 128 + i_row;
                    float pg[kMx4Chunk], pu[kMx4Chunk];
#pragma unroll
                    for (int j = 0; j < kMx4Chunk; ++j) {
                        pg[j] = j < n ? __ldcg(p + (col + j) * 128) : 0.f;
                        pu[j] = j < n ? __ldcg(p + (NT + col + j) * 128) : 0.f;
                    }
#pragma unroll
                    for (int j = 0; j < kMx4Chunk; ++j) {
                        g[j] += pg[j];
                        u[j] += pu[j];
                    }
                }
                finish(t, col, n, g, u);
            }
        }
    }

    if (PAIR) {
        // The other CTA may raise this one's abort flag at any time, so every thread
        // acts on one snapshot taken after the roles have finished.
        __syncthreads();
        if (threadIdx.x == 0) s_misc[1] = *abort_flag;
        if (warp == 1 && rank == 0) {
            if (elect_one()) umma_commit_pair(smem_u32(drain_bar));   // every MMA has completed
            __syncwarp();
            volatile int never = 0;
            mbar_wait(drain_bar, 0, &never);
        }
        __syncthreads();
        if (s_misc[1]) {
            // let this CTA's copies in flight land before its shared memory is released
            const unsigned long long t0 = global_timer_ns();
            while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
        }
        tc_fence_before();
        cluster_sync_all();   // nothing of the other CTA still reaches into this one
        if (warp == 1) {
            tc_fence_after();
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kMx4TmemCols)
                         : "memory");
        }
        return;
    }
    __syncthreads();
    if (*abort_flag) {
        if (warp == 1) {
            if (elect_one()) umma_commit(drain_bar);
            __syncwarp();
            volatile int never = 0;
            mbar_wait(drain_bar, 0, &never);
        }
        const unsigned long long t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kMx4TmemCols)
                     : "memory");
    }
}

}  // namespace pdx
