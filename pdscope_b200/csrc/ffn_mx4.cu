// Grouped SwiGLU experts on MXFP4 weights: y[p] = Wd (silu(Wg x) * (Wu x)) for
// every packed row p, weights dequantised exactly, sums and h in FP32, one
// rounding to BF16 at the end.  One warp per output value pair.
#include "ffn_gemv.cu"
#include "mxfp4.cu"

namespace pdx {

// Expert weights: slot s holds, from codes + s * code_stride, gate [Ip, Hp/2],
// up [Ip, Hp/2] and down [Hp, Ip/2] code bytes (Hp, Ip: H, I rounded up to
// 128, padding zero), and from scales + s * scale_stride their scales as tiles
// of 128 rows x 128 columns, 512 bytes each, row tiles outermost: byte
// (r % 32) * 16 + (r / 32) * 4 + c / 32 of a tile is the scale of row r,
// columns c .. c + 31.
struct Mx4Slab {
    const uint8_t* codes;
    const uint8_t* scales;
    int64_t code_stride, scale_stride, num_slots;
    const int32_t* slot_of_expert;
};

__device__ __forceinline__ int64_t mx4_tile_scale(int r, int c, int cols) {
    return (static_cast<int64_t>(r >> 7) * (cols >> 7) + (c >> 7)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 +
           ((c >> 5) & 3);
}

// Expert of packed row p and its weight slot (flagged slots read slot 0).
__device__ __forceinline__ int64_t mx4_row_slot(const Mx4Slab& w, const int32_t* offsets, const int32_t* active,
                                                int p) {
    int lo = 0, hi = active[0] - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (offsets[active[1 + mid]] <= p) lo = mid; else hi = mid - 1;
    }
    const int e = active[1 + lo];
    if (p < offsets[e] || p >= offsets[e + 1]) return -1;   // a row of no active expert
    const int64_t slot = w.slot_of_expert ? w.slot_of_expert[e] : e;
    if (slot < 0 || slot >= w.num_slots) {
        raise_error(PDX_DEVERR_BAD_SLOT);
        return 0;
    }
    return slot;
}

__global__ void __launch_bounds__(256) k_mx4_gateup(const uint16_t* __restrict__ x, const int32_t* __restrict__ tokens,
                                                    int T, const int32_t* __restrict__ offsets,
                                                    const int32_t* __restrict__ active, Mx4Slab w, int rows, int H,
                                                    int I, int Hp, int Ip, float* __restrict__ h) {
    griddep_wait();
    griddep_launch();
    const int p = static_cast<int>(blockIdx.x);
    const int64_t slot = mx4_row_slot(w, offsets, active, p);
    if (slot < 0) return;
    int t = tokens ? tokens[p] : p;
    if (t < 0 || t >= T) {
        raise_error(PDX_DEVERR_BAD_EXPERT);
        t = 0;
    }
    const uint8_t* gc = w.codes + slot * w.code_stride;
    const uint8_t* uc = gc + static_cast<int64_t>(Ip) * Hp / 2;
    const uint8_t* gs = w.scales + slot * w.scale_stride;
    const uint8_t* us = gs + static_cast<int64_t>(Ip) * Hp / 32;
    for (int i = static_cast<int>(blockIdx.y) * 8 + static_cast<int>(threadIdx.x >> 5); i < I; i += 8 * gridDim.y) {
        float g = 0.f, u = 0.f;
        for (int k = static_cast<int>(lane_id()) * 8; k < H; k += 256) {
            float xv[8], gv[8], uv[8];
            load8<bf16, true>(reinterpret_cast<const bf16*>(x) + static_cast<int64_t>(t) * H + k, xv);
            const int64_t at = (static_cast<int64_t>(i) * Hp + k) / 2, sc = mx4_tile_scale(i, k, Hp);
            e2m1x8_to_float(*reinterpret_cast<const uint32_t*>(gc + at), gv);
            e2m1x8_to_float(*reinterpret_cast<const uint32_t*>(uc + at), uv);
            float a = 0.f, b = 0.f;
            for (int j = 0; j < 8; ++j) {
                a += xv[j] * gv[j];
                b += xv[j] * uv[j];
            }
            g += a * mx_scale(gs[sc]);
            u += b * mx_scale(us[sc]);
        }
        g = warp_sum(g);
        u = warp_sum(u);
        if (lane_id() == 0) h[static_cast<int64_t>(p) * I + i] = g / (1.f + expf(-g)) * u;
    }
}

__global__ void __launch_bounds__(256) k_mx4_down(const float* __restrict__ h, const int32_t* __restrict__ offsets,
                                                  const int32_t* __restrict__ active, Mx4Slab w, int rows, int H, int I,
                                                  int Hp, int Ip, uint16_t* __restrict__ y) {
    griddep_wait();
    griddep_launch();
    const int p = static_cast<int>(blockIdx.x);
    const int64_t slot = mx4_row_slot(w, offsets, active, p);
    if (slot < 0) return;
    const uint8_t* dc = w.codes + slot * w.code_stride + static_cast<int64_t>(Ip) * Hp;
    const uint8_t* ds = w.scales + slot * w.scale_stride + static_cast<int64_t>(Ip) * Hp / 16;
    for (int c = static_cast<int>(blockIdx.y) * 8 + static_cast<int>(threadIdx.x >> 5); c < H; c += 8 * gridDim.y) {
        float acc = 0.f;
        for (int k = static_cast<int>(lane_id()) * 8; k < I; k += 256) {
            float hv[8], dv[8];
            load8<float, true>(h + static_cast<int64_t>(p) * I + k, hv);
            e2m1x8_to_float(*reinterpret_cast<const uint32_t*>(dc + (static_cast<int64_t>(c) * Ip + k) / 2), dv);
            float a = 0.f;
            for (int j = 0; j < 8; ++j) a += hv[j] * dv[j];
            acc += a * mx_scale(ds[mx4_tile_scale(c, k, Ip)]);
        }
        acc = warp_sum(acc);
        if (lane_id() == 0) y[static_cast<int64_t>(p) * H + c] = f2bits(acc);
    }
}

}  // namespace pdx
