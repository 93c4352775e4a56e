// Launch functions of the vocabulary objectives (objectives.cu, top_logits.cu, preference.cu), called by
// their PyTorch side (objectives_torch.cpp), which checks the arguments. Nothing here needs PyTorch.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace me {

constexpr int64_t kIgnoreToken = -100;  // the target of an untrained token
constexpr int kMaxTop = 256;            // most teacher entries / top logits of a row
// Most columns of a row. The kernels count them in 32 bits, and a loop that steps by a block's threads (or by their
// vectors: 256 times 8 columns) ends up to 2048 past the row's end.
constexpr int64_t kMaxColumns = INT32_MAX - 4096;

enum class LogitType : int { kBF16 = 0, kF16 = 1, kF32 = 2 };

// N rows of V raw logits, `stride` elements apart; cap <= 0: no softcap.
struct Logits {
  const void* data;
  int64_t stride, N, V;
  LogitType type;
  float cap;
};
// Where their gradient goes (the logits' type; it may be the logits themselves).
struct Gradient {
  void* data;
  int64_t stride;
};

// One number a row, `step` apart (0: one for all).
struct RowValues {
  const float* data;
  int64_t step;
};

// The teacher's records: k entries a row; lse and weight may be null.
struct TeacherArgs {
  const int64_t* ids;
  const float* top;
  const float* lse;
  const float* weight;
  int k;
  float temp;
};

void launch_logprob_fwd(const Logits& x, const int64_t* target, float* logp, float2* stats, cudaStream_t stream);
void launch_logprob_bwd(const Logits& x, const int64_t* target, const float2* stats, RowValues g, Gradient out,
                        cudaStream_t stream);
// What launch_teacher() leaves for the other three: N k entries and N rows, 16-byte aligned.
constexpr int kEntryBytes = 16, kTeacherRowBytes = 32;
void launch_teacher(const Logits& x, const TeacherArgs& teacher, void* entries, void* rows, cudaStream_t stream);
void launch_distill_fwd(const Logits& x, const TeacherArgs& teacher, const void* entries, const void* rows, float* loss,
                        float4* stats, cudaStream_t stream);
// value and gradient of sum(loss) in one launch
void launch_distill_grad(const Logits& x, const TeacherArgs& teacher, const void* entries, const void* rows, float* loss,
                         Gradient out, cudaStream_t stream);
// g: one coefficient a row
void launch_distill_bwd(const Logits& x, const TeacherArgs& teacher, const void* entries, const void* rows,
                        const float4* stats, RowValues g, Gradient out, cudaStream_t stream);
void launch_top_logits(const Logits& x, int k, float temp, float* values, int64_t* ids, float* lse,
                       cudaStream_t stream);

struct PairArgs {
  const float *logp, *ref;  // ref may be null
  const int64_t* target;    // or null: every token is trained
  const void* cu;           // [2 pairs + 1], int32 or int64
  bool cu64;
  int64_t tokens, pairs;
  int kind;  // 0 sigmoid, 1 hinge, 2 ipo
  float beta, smooth, scale;
};
void launch_preference(const PairArgs& a, float* loss, float2* rewards, float* grad, cudaStream_t stream);
// out_t = grad_t * g of the token's pair
void launch_preference_scale(const float* grad, const float* g, const void* cu, bool cu64, int64_t tokens, int64_t pairs,
                             float* out, cudaStream_t stream);

}  // namespace me
