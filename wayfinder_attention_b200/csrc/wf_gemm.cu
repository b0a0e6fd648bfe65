// The product with an epilogue (wf_gemm_kernel.cuh): tile shapes, split depths and launches.
#include "wf_gemm_kernel.cuh"

namespace wf {
namespace {

// Adds the parts of a split depth and applies the epilogue: a thread takes 4 columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) gemm_join_kernel(const float* partial, int splits, int64_t pitch, int64_t M,
                                                        int64_t N, GemmEpilogue o) {
  using Z = typename Kept<T>::type;
  pdl_wait();
  const int64_t groups = pitch / 4, total = M * groups;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / groups, n = i % groups * 4;
    const int live = (int)min((int64_t)4, N - n);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
      const float4 f = *reinterpret_cast<const float4*>(partial + ((int64_t)s * M + m) * pitch + n);
      v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
    }
    if (o.factor)
      for (int j = 0; j < 4; ++j) v[j] *= *o.factor;
    if (o.bias)
      for (int j = 0; j < live; ++j) v[j] += to_f32(static_cast<const T*>(o.bias)[n + j]);
    if (o.z)
      for (int j = 0; j < live; ++j)
        static_cast<Z*>(o.z)[m * o.z_stride + n + j] = from_f32<Z>(kept_z(o.act, v[j]));
    activate_all<T, 4>(o.act, v);
    if (o.residual)
      for (int j = 0; j < live; ++j) v[j] += to_f32(static_cast<const T*>(o.residual)[m * o.r_stride + n + j]);
    for (int j = 0; j < live; ++j) static_cast<T*>(o.y)[m * o.y_stride + n + j] = from_f32<T>(v[j]);
  }
}

// Tile shape and depth shares: the least of an estimate over the shapes there are.  A
// unit's time is its stages of depth at the rate the shape can take them plus its
// accumulator's way out; units run in waves.
constexpr Shape kShapes[] = {{256, 2, 560, 0}, {128, 2, 400, 1700}, {128, 1, 540, 0}, {64, 1, 400, 1300}};
constexpr int kMinShare = 4;  // stages of depth a share has at least
Plan plan_of(int64_t M, int64_t N, int64_t K, int pieces, int turns) {
  Plan best{};
  double least = 0;
  for (const Shape& s : kShapes) {
    if (pieces > 1 && !s.cycles3) continue;
    Plan p{};
    p.shape = s;
    p.k_blocks = (int)((K + kBK - 1) / kBK) * turns;
    const int64_t tn = (N + s.bn - 1) / s.bn, tm = (M + kBM * s.cg - 1) / (kBM * s.cg);
    p.tiles_n = (int)tn;
    p.tiles = (int)(tn * tm);
    const int slots = kSms / s.cg;
    for (int splits = 1; splits <= kMaxSplits && (splits == 1 || p.k_blocks / splits >= kMinShare); ++splits) {
      if (splits > 1 && (int64_t)p.tiles * splits > 2 * slots) break;  // most shapes look at one split
      const int64_t waves = ((int64_t)p.tiles * splits + slots - 1) / slots;
      const int64_t deep = (p.k_blocks + splits - 1) / splits;
      // partials go through L2 twice, and joining them is a launch
      const double join = splits > 1 ? 4000 + 8.0 * splits * M * N / 4000 : 0;
      const double t = (double)waves * (deep * (pieces > 1 ? s.cycles3 : s.cycles) + 4 * s.bn) + join;
      if (best.splits == 0 || t < least) {
        least = t;
        best = p;
        best.splits = best.layers = splits;
      }
    }
  }
  return best;
}

template <typename T, bool PIECES, class E = Finish>
int launch_shape(const GemmProblem& g, const GemmEpilogue& out, const Plan& plan, cudaStream_t stream) {
  const Shape& s = plan.shape;
  if constexpr (!PIECES) {
    if (s.bn == 256) return launch_tile<T, 256, 2, PIECES>(g, out, plan, E{}, stream);
    if (s.bn == 128 && s.cg == 1) return launch_tile<T, 128, 1, PIECES>(g, out, plan, E{}, stream);
  }
  if (s.cg == 2) return launch_tile<T, 128, 2, PIECES>(g, out, plan, E{}, stream);
  return launch_tile<T, 64, 1, PIECES>(g, out, plan, E{}, stream);
}

template <typename T, bool PIECES>
int launch_type(const GemmProblem& g, cudaStream_t stream) {
  const Plan plan = plan_of(g.M, g.N, g.K, g.pieces, g.turns);
  if (plan.splits == 1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      if (g.out.factor) return launch_shape<T, PIECES, FinishByFactor>(g, g.out, plan, stream);
    return launch_shape<T, PIECES>(g, g.out, plan, stream);
  }
  GemmEpilogue parts{};
  parts.y = g.ws;
  parts.y_stride = round8(g.N);
  if (int rc = launch_shape<float, PIECES>(g, parts, plan, stream)) return rc;
  const int64_t work = (g.M * (parts.y_stride / 4) + 255) / 256;
  return (int)launch_pdl(gemm_join_kernel<T>, dim3((unsigned)std::min<int64_t>(work, 8 * kSms)), dim3(256), 0, stream,
                         static_cast<const float*>(g.ws), plan.splits, parts.y_stride, g.M, g.N, g.out);
}

}  // namespace

size_t gemm_workspace_bytes(int64_t M, int64_t N, int64_t K, int pieces, int turns) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan p = plan_of(M, N, K, pieces, turns);
  return p.splits > 1 ? (size_t)p.splits * M * round8(N) * sizeof(float) : 0;
}

int launch_gemm(const GemmProblem& g, cudaStream_t stream) {
  if (g.M == 0 || g.N == 0) return 0;
  if (g.out.factor && g.out_dtype != kBF16) return -1;  // nothing asks for it
  if (g.out_dtype == kBF16) return launch_type<__nv_bfloat16, false>(g, stream);
  if (g.out_dtype == kF16) return launch_type<__half, false>(g, stream);
  return g.pieces == 1 ? launch_type<float, false>(g, stream) : launch_type<float, true>(g, stream);
}

}  // namespace wf
