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

constexpr int kBnMaxH = 8192;      // eight values per thread, 1024 threads

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

// Sum over the CTA in a fixed order.  Successive calls alternate between two
// halves of red[64], so one barrier a call is enough.
__device__ __forceinline__ float bn_block_sum(float v, float* red, int& turn) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    const int warps = static_cast<int>(blockDim.x >> 5);
    if (warps == 1) return v;
    float* r = red + 32 * turn;
    turn ^= 1;
    if (lane_id() == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    v = static_cast<int>(lane_id()) < warps ? r[lane_id()] : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// A thread's eight values of a row of H: VEC, the aligned eight from 8 * tid;
// else every blockDim-th value from tid (any H and alignment).  Values past H
// read as 0 and are not written.
template <bool VEC>
struct BnPlace {
    int H, first, step;
    __device__ explicit BnPlace(int h)
        : H(h), first(static_cast<int>(threadIdx.x) * (VEC ? 8 : 1)), step(VEC ? 1 : static_cast<int>(blockDim.x)) {}
    __device__ __forceinline__ int col(int i) const { return first + i * step; }
    __device__ __forceinline__ bool in(int i) const { return VEC ? first < H : col(i) < H; }
};

// Raw values, loaded early and converted where they are used.
template <bool VEC, typename T>
struct BnRaw;
template <>
struct BnRaw<true, uint16_t> {
    uint4 q;
    __device__ __forceinline__ void load(const BnPlace<true>& at, const uint16_t* p) {
        q = make_uint4(0, 0, 0, 0);
        if (at.in(0)) q = *reinterpret_cast<const uint4*>(p + at.first);
    }
    __device__ __forceinline__ float get(int i) const {
        const uint32_t w = i < 2 ? q.x : (i < 4 ? q.y : (i < 6 ? q.z : q.w));
        return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
    }
};
template <>
struct BnRaw<true, float> {
    float4 a, b;
    __device__ __forceinline__ void load(const BnPlace<true>& at, const float* p) {
        a = b = make_float4(0.f, 0.f, 0.f, 0.f);
        if (at.in(0)) {
            a = reinterpret_cast<const float4*>(p + at.first)[0];
            b = reinterpret_cast<const float4*>(p + at.first)[1];
        }
    }
    __device__ __forceinline__ float get(int i) const {
        const float4& v = i < 4 ? a : b;
        return (i & 3) == 0 ? v.x : ((i & 3) == 1 ? v.y : ((i & 3) == 2 ? v.z : v.w));
    }
};
template <>
struct BnRaw<false, uint16_t> {
    uint16_t v[8];
    __device__ __forceinline__ void load(const BnPlace<false>& at, const uint16_t* p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = at.in(i) ? p[at.col(i)] : static_cast<uint16_t>(0);
    }
    __device__ __forceinline__ float get(int i) const { return bits2f(v[i]); }
};
template <>
struct BnRaw<false, float> {
    float v[8];
    __device__ __forceinline__ void load(const BnPlace<false>& at, const float* p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = at.in(i) ? p[at.col(i)] : 0.f;
    }
    __device__ __forceinline__ float get(int i) const { return v[i]; }
};

template <bool VEC>
__device__ __forceinline__ void bn_store(const BnPlace<VEC>& at, uint16_t* p, const float* v) {
    if (VEC) {
        if (!at.in(0)) return;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = static_cast<uint32_t>(f2bits(v[2 * i])) | (static_cast<uint32_t>(f2bits(v[2 * i + 1])) << 16);
        *reinterpret_cast<uint4*>(p + at.first) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at.in(i)) p[at.col(i)] = f2bits(v[i]);
    }
}
template <bool VEC>
__device__ __forceinline__ void bn_store(const BnPlace<VEC>& at, float* p, const float* v) {
    if (VEC) {
        if (!at.in(0)) return;
        reinterpret_cast<float4*>(p + at.first)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p + at.first)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at.in(i)) p[at.col(i)] = v[i];
    }
}

// Normalise the row held in v (values past H are 0 and stay so).
template <bool VEC>
__device__ __forceinline__ void bn_norm(float (&v)[8], int how, bool weighted, const BnRaw<VEC, uint16_t>& w,
                                        const BnPlace<VEC>& at, float eps, float* red, int& turn) {
    if (how == PDX_NORM_NONE) return;
    const float inv_h = 1.0f / static_cast<float>(at.H);
    if (how == PDX_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
        const float mean = bn_block_sum(s, red, turn) * inv_h;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at.in(i)) v[i] -= mean;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) q += v[i] * v[i];
    const float inv = rsqrtf(bn_block_sum(q, red, turn) * inv_h + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= weighted ? inv * w.get(i) : inv;
}

// One CTA per row, eight values a thread, at most MAXT threads.  EARLY (few rows,
// where the latency of a row counts): every load that does not depend on a
// reduction is issued before the first one, so a row costs one trip to memory
// and up to four block reductions.  Otherwise rows hide each other's latency and
// what counts is how many fit an SM: the weights (and beside expert rows the gate)
// are loaded where they are used, at no more than 42 registers (48 warps an SM).
template <typename RES, bool COMBINE, bool VEC, int MAXT, bool EARLY>
__global__ void __launch_bounds__(MAXT, EARLY || MAXT == 1024 ? 1 : 1536 / MAXT) k_block_norm(BlockNormArgs a) {
    // expert rows loaded together; any-alignment rows take a register per value
    constexpr int kBatch = !VEC ? 2 : (EARLY && MAXT < 1024 ? 8 : 4);
    griddep_wait();
    griddep_launch();
    __shared__ float red[64];
    __shared__ int s_row[32];
    __shared__ float s_w[32];
    const int64_t t = blockIdx.x;
    const int H = a.H;
    const BnPlace<VEC> at(H);
    int turn = 0;
    BnRaw<VEC, RES> res;
    BnRaw<VEC, uint16_t> yr, gate, post_w, pre_w;
    res.load(at, static_cast<const RES*>(a.residual) + t * H);
    if (!COMBINE && a.y) yr.load(at, a.y + t * H);
    float gate_one = 1.f;
    const bool gate_rowwise = a.gate && a.gate_col == 1;
    auto load_gate = [&]() {
        if (gate_rowwise)
            gate.load(at, a.gate + t * a.gate_row);
        else if (a.gate && a.gate_col == 0)
            gate_one = bits2f(a.gate[t * a.gate_row]);
    };
    if (EARLY || !COMBINE) load_gate();
    if (EARLY) {
        if (a.post_weight) post_w.load(at, a.post_weight);
        if (VEC && a.pre_weight) pre_w.load(at, a.pre_weight);
    }
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
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
        // FP32 sum in slot order
        for (int s0 = 0; s0 < a.k; s0 += kBatch) {
            BnRaw<VEC, uint16_t> r[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (s0 + j < a.k && s_row[s0 + j] >= 0) r[j].load(at, a.y + static_cast<int64_t>(s_row[s0 + j]) * H);
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (s0 + j < a.k && s_row[s0 + j] >= 0)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] += r[j].get(i) * s_w[s0 + j];
        }
    } else if (a.y) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = yr.get(i);
    }
    if (!EARLY && a.post_weight) post_w.load(at, a.post_weight);
    if (COMBINE || a.y) bn_norm<VEC>(v, a.post, a.post_weight != nullptr, post_w, at, a.eps, red, turn);
    if (!EARLY && COMBINE) load_gate();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float g = gate_one;
        if (gate_rowwise)
            g = gate.get(i);
        else if (a.gate && a.gate_col > 1 && at.in(i))
            g = bits2f(a.gate[t * a.gate_row + at.col(i) * a.gate_col]);
        if (a.gate && a.gate_sigmoid) g = __fdividef(1.0f, 1.0f + expf(-g));   // approximate reciprocal: 1 ulp
        v[i] = a.residual_scale * res.get(i) + a.block_scale * (a.gate ? g * v[i] : v[i]);
        if (!at.in(i)) v[i] = 0.f;
    }
    if (a.stream) bn_store<VEC>(at, static_cast<RES*>(a.stream) + t * H, v);
    if (!a.normed) return;
    if (!(EARLY && VEC) && a.pre_weight) pre_w.load(at, a.pre_weight);
    bn_norm<VEC>(v, a.pre, a.pre_weight != nullptr, pre_w, at, a.eps, red, turn);
    bn_store<VEC>(at, a.normed + t * H, v);
}

}  // namespace pdx
