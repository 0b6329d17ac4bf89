// The norms around a block in one pass: the norm after the block, its gate and
// the residual scale, and the norm before the next block.  Per row, in FP32,
//   y = block output, or sum_s w[t, s] * rows[inverse[t*k + s]]   (COMBINE)
//   z = post(y) * post_weight
//   s = residual_scale * r + block_scale * act(gate) * z          -> stream
//   n = pre(s) * pre_weight                                       -> normed
// with post, pre one of none, rms (v / sqrt(mean v^2 + eps)) and layer
// ((v - mean) / sqrt(var + eps), population variance).  s feeds the second
// norm unrounded; each output is rounded once.
// Bound by HBM (y or the k rows, r, s, n once each) or, for a few rows, by the
// chain load -> up to four block reductions -> store.  The row stays in
// registers between the reductions, so nothing is read twice.
#include "pdx_common.cuh"

namespace pdx {

constexpr int kBnThreads = 256;
constexpr int kBnMaxH = 8192;

struct BlockNormArgs {
    const uint16_t* y;            // [T, H], or the expert rows [y_rows, H] (COMBINE)
    const uint16_t* weights;      // [T, k] (COMBINE)
    const int32_t* inverse;       // [T, k] (COMBINE)
    int k, y_rows;
    const void* residual;         // [T, H] BF16 or FP32
    const uint16_t* post_weight;  // [H] or NULL
    const uint16_t* pre_weight;   // [H] or NULL
    const uint16_t* gate;         // NULL = 1
    int64_t gate_row, gate_col;   // element strides of the gate (0 = broadcast)
    int gate_sigmoid;
    int post, pre;
    float residual_scale, block_scale, eps;
    int H;
    void* stream;                 // residual's type, or NULL
    uint16_t* normed;             // or NULL
};

__device__ __forceinline__ float bn_block_sum(float v, float* red) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    __syncthreads();  // red[] free from the previous reduction
    if (lane_id() == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float tot = 0.f;
#pragma unroll
    for (int w = 0; w < kBnThreads / 32; ++w) tot += red[w];
    return tot;
}

template <int VEC>
__device__ __forceinline__ void bn_load(const uint16_t* p, float* v) {
    if (VEC == 8) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
        v[0] = bits2f(p[0]);
    }
}

template <int VEC>
__device__ __forceinline__ void bn_load(const float* p, float* v) {
    if (VEC == 8) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        v[0] = p[0];
    }
}

template <int VEC>
__device__ __forceinline__ void bn_store(uint16_t* p, const float* v) {
    if (VEC == 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = static_cast<uint32_t>(f2bits(v[2 * i])) | (static_cast<uint32_t>(f2bits(v[2 * i + 1])) << 16);
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        p[0] = f2bits(v[0]);
    }
}

template <int VEC>
__device__ __forceinline__ void bn_store(float* p, const float* v) {
    if (VEC == 8) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        p[0] = v[0];
    }
}

// Normalise this thread's values of the row in place (values past H stay 0).
template <int VEC, int CH>
__device__ __forceinline__ void bn_norm(float (&v)[CH * VEC], int how, const uint16_t* __restrict__ weight, int H,
                                        float eps, float* red) {
    if (how == PDX_NORM_NONE) return;
    const float inv_h = 1.0f / static_cast<float>(H);
    float mean = 0.f;
    if (how == PDX_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < CH * VEC; ++i) s += v[i];
        mean = bn_block_sum(s, red) * inv_h;
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j)
        if ((static_cast<int>(threadIdx.x) + j * kBnThreads) * VEC < H)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[j * VEC + i] -= mean;
                q += v[j * VEC + i] * v[j * VEC + i];
            }
    const float inv = rsqrtf(bn_block_sum(q, red) * inv_h + eps);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = (static_cast<int>(threadIdx.x) + j * kBnThreads) * VEC;
        if (c < H) {
            float w[VEC];
            if (weight) bn_load<VEC>(weight + c, w);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[j * VEC + i] *= weight ? inv * w[i] : inv;
        }
    }
}

// One CTA per row; thread i owns the VEC values from (i + 256 j) * VEC, j < CH.
// VEC = 8 needs H % 8 == 0 and 16-byte aligned rows, VEC = 1 takes any H.
template <typename RES, bool COMBINE, int VEC, int CH>
__global__ void __launch_bounds__(kBnThreads) k_block_norm(BlockNormArgs a) {
    griddep_wait();
    griddep_launch();
    __shared__ float red[kBnThreads / 32];
    __shared__ int s_row[32];
    __shared__ float s_w[32];
    const int64_t t = blockIdx.x;
    const int H = a.H;
    if (COMBINE) {
        if (threadIdx.x < static_cast<unsigned>(a.k)) {
            int row = a.inverse[t * a.k + threadIdx.x];
            float w = bits2f(a.weights[t * a.k + threadIdx.x]);
            if (row < 0 || row >= a.y_rows) {
                raise_error(PDX_DEVERR_BAD_EXPERT);
                row = -1;
            }
            s_row[threadIdx.x] = row;
            s_w[threadIdx.x] = w;
        }
        __syncthreads();
    }
    float v[CH * VEC];
#pragma unroll
    for (int i = 0; i < CH * VEC; ++i) v[i] = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = (static_cast<int>(threadIdx.x) + j * kBnThreads) * VEC;
        if (c < H) {
            if (COMBINE) {
                for (int s = 0; s < a.k; ++s) {
                    if (s_row[s] < 0) continue;
                    float r[VEC];
                    bn_load<VEC>(a.y + static_cast<int64_t>(s_row[s]) * H + c, r);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[j * VEC + i] += r[i] * s_w[s];
                }
            } else if (a.y) {
                bn_load<VEC>(a.y + t * H + c, &v[j * VEC]);
            }
        }
    }
    if (COMBINE || a.y) bn_norm<VEC, CH>(v, a.post, a.post_weight, H, a.eps, red);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = (static_cast<int>(threadIdx.x) + j * kBnThreads) * VEC;
        if (c < H) {
            float r[VEC], g[VEC];
            bn_load<VEC>(static_cast<const RES*>(a.residual) + t * H + c, r);
            if (a.gate) {
                const uint16_t* gp = a.gate + t * a.gate_row;
                if (a.gate_col == 1) {
                    bn_load<VEC>(gp + c, g);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) g[i] = bits2f(gp[(c + i) * a.gate_col]);
                }
                if (a.gate_sigmoid)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) g[i] = 1.0f / (1.0f + expf(-g[i]));
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float z = a.block_scale * (a.gate ? g[i] * v[j * VEC + i] : v[j * VEC + i]);
                v[j * VEC + i] = a.residual_scale * r[i] + z;
            }
            if (a.stream) bn_store<VEC>(static_cast<RES*>(a.stream) + t * H + c, &v[j * VEC]);
        }
    }
    if (!a.normed) return;
    bn_norm<VEC, CH>(v, a.pre, a.pre_weight, H, a.eps, red);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = (static_cast<int>(threadIdx.x) + j * kBnThreads) * VEC;
        if (c < H) bn_store<VEC>(a.normed + t * H + c, &v[j * VEC]);
    }
}

}  // namespace pdx
