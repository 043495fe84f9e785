// C entry points of the block operators (include/eg2_hip.h): the checks of
// their records and the launches.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "eg2_block.hpp"
#include "eg2_hip.h"

namespace {

constexpr int kInvalid = (int)hipErrorInvalidValue;
constexpr unsigned kMost = 1u << 24;

bool is_activation_type(unsigned t) { return t == EG2_TYPE_F32 || t == EG2_TYPE_F16 || t == EG2_TYPE_BF16; }
unsigned size_of(unsigned t) { return t == EG2_TYPE_F32 ? 4u : 2u; }
bool on(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// rows * stride and heads * stride stay far inside 64 bits.
bool small(uint64_t stride) { return stride < (uint64_t)1 << 31; }

bool weights_fit(unsigned type, unsigned weight_type, const void* w, unsigned k, uint64_t ldw) {
  if (!w || !small(ldw)) return false;
  if (weight_type == EG2_TYPE_Q8_0) return on(w, 2) && k % 32 == 0 && ldw % 32 == 0;
  if (!is_activation_type(weight_type) || (type != EG2_TYPE_F32 && weight_type != type)) return false;
  return on(w, size_of(weight_type));
}
bool sizes_fit(unsigned n, unsigned k, unsigned m, unsigned type, unsigned act) {
  return n > 0 && k > 0 && m > 0 && n <= kMost && k <= kMost && m <= kMost && (uint64_t)n * m <= (uint64_t)1 << 32 &&
         is_activation_type(type) && act <= EG2_ACT_RELU;
}

bool valid(const eg2_linear_args& a) {
  if (!sizes_fit(a.n, a.k, a.m, a.type, a.act) || !a.y || !a.x) return false;
  const unsigned size = size_of(a.type);
  if (!on(a.y, size) || !on(a.x, size) || !on(a.bias, 4) || !on(a.residual, size)) return false;
  if (!small(a.ldx) || !small(a.ldy) || a.ldy < a.m || (a.residual && !small(a.ldr))) return false;
  if (a.residual == a.y && a.ldr != a.ldy) return false;
  return weights_fit(a.type, a.weight_type, a.weight, a.k, a.ldw);
}

bool valid(const eg2_linear_gated_args& a) {
  if (!sizes_fit(a.n, a.k, a.m, a.type, a.act) || !a.y || !a.x) return false;
  const unsigned size = size_of(a.type);
  if (!on(a.y, size) || !on(a.x, size) || !on(a.gate_bias, 4) || !on(a.up_bias, 4)) return false;
  if (!small(a.ldx) || !small(a.ldy) || a.ldy < a.m) return false;
  return weights_fit(a.type, a.weight_type, a.gate, a.k, a.ldw) && weights_fit(a.type, a.weight_type, a.up, a.k, a.ldw);
}

bool valid(const eg2_heads_norm_rope_args& a) {
  if (!is_activation_type(a.type) || a.rows == 0 || a.rows > kMost || a.d < 2 || a.d > 512 || a.d % 2 != 0 ||
      a.rotary > a.d || a.rotary % 2 != 0 || a.q_heads == 0 || a.q_heads > 4096 || a.k_heads > 4096 ||
      a.q_heads + a.k_heads > 4096 || (uint64_t)a.rows * (a.q_heads + a.k_heads) > (uint64_t)1 << 25)
    return false;
  const unsigned size = size_of(a.type);
  if (!a.q || !a.q_out || !on(a.q, size) || !on(a.q_out, size) || !small(a.q_row) || !small(a.q_head) ||
      !small(a.q_out_row) || !small(a.q_out_head))
    return false;
  if (a.k_heads && (!a.k || !a.k_out || !on(a.k, size) || !on(a.k_out, size) || !small(a.k_row) || !small(a.k_head) ||
                    !small(a.k_out_row) || !small(a.k_out_head)))
    return false;
  if (a.q == a.q_out && (a.q_row != a.q_out_row || a.q_head != a.q_out_head)) return false;
  if (a.k_heads && a.k == a.k_out && (a.k_row != a.k_out_row || a.k_head != a.k_out_head)) return false;
  if (!on(a.q_weight, 4) || !on(a.k_weight, 4)) return false;
  if (a.rotary && (!a.table || !a.pos || !on(a.table, 4) || !on(a.pos, 4) || a.table_rows == 0)) return false;
  return true;
}

// What the workspace follows from.
bool valid_sizes(const eg2_window_attention_args& a) {
  return is_activation_type(a.type) && a.batch > 0 && a.batch <= 65535 && a.rows > 0 && a.rows <= 1u << 27 &&
         a.key_rows > 0 && a.key_rows <= 1u << 30 && a.kv_heads > 0 && a.heads > 0 && a.heads <= 4096 &&
         a.heads % a.kv_heads == 0 && a.d >= 8 && a.d <= 256 && a.d % 8 == 0 &&
         (uint64_t)a.rows * a.heads <= (uint64_t)1 << 27 && (uint64_t)a.batch * a.kv_heads <= (uint64_t)1 << 22;
}
bool valid(const eg2_window_attention_args& a) {
  if (!valid_sizes(a) || !a.q_offsets || !a.k_offsets || !on(a.q_offsets, 4) || !on(a.k_offsets, 4) ||
      !on(a.k_lengths, 4) || !(std::fabs(a.scale) <= 0x1p127f))
    return false;
  const unsigned per16 = 16 / size_of(a.type);
  auto rows_fit = [&](const void* p, uint64_t row, uint64_t head) {
    return p && on(p, 16) && row % per16 == 0 && head % per16 == 0 && small(row) && small(head);
  };
  if (!rows_fit(a.q, a.q_row, a.q_head) || !rows_fit(a.k, a.k_row, a.k_head) || !rows_fit(a.v, a.v_row, a.v_head) ||
      !rows_fit(a.out, a.out_row, a.out_head))
    return false;
  const uint64_t need = eg2::block::window_attention_workspace(a);
  return need == 0 || (a.workspace && on(a.workspace, 16) && a.workspace_bytes >= need);
}

hipError_t launch_linear(const eg2::block::Linear& p, unsigned type, unsigned weight_type, bool gated, hipStream_t st) {
  switch (type) {
    case EG2_TYPE_F32:
      return eg2::block::launch_linear_f32(p, weight_type, gated, st);
    case EG2_TYPE_F16:
      return eg2::block::launch_linear_f16(p, weight_type, gated, st);
    default:
      return eg2::block::launch_linear_bf16(p, weight_type, gated, st);
  }
}
hipError_t launch(const eg2_linear_args& a, hipStream_t st) {
  return launch_linear({a.y, a.x, {a.weight, nullptr}, {a.bias, nullptr}, a.residual, a.ldx, a.ldw, a.ldy, a.ldr, a.n, a.k,
                        a.m, a.act},
                       a.type, a.weight_type, false, st);
}
hipError_t launch(const eg2_linear_gated_args& a, hipStream_t st) {
  return launch_linear({a.y, a.x, {a.gate, a.up}, {a.gate_bias, a.up_bias}, nullptr, a.ldx, a.ldw, a.ldy, 0, a.n, a.k, a.m,
                        a.act},
                       a.type, a.weight_type, true, st);
}
hipError_t launch(const eg2_heads_norm_rope_args& a, hipStream_t st) { return eg2::block::launch_heads_norm_rope(a, st); }
hipError_t launch(const eg2_window_attention_args& a, hipStream_t st) { return eg2::block::launch_window_attention(a, st); }

template <class Args>
int checked(const Args* args, void* stream) {
  if (!args || !valid(*args)) return kInvalid;
  return (int)launch(*args, reinterpret_cast<hipStream_t>(stream));
}

}  // namespace

extern "C" {

int eg2_hip_linear(const eg2_linear_args* args, void* stream) {
  return checked(args, stream);
}

int eg2_hip_linear_gated(const eg2_linear_gated_args* args, void* stream) {
  return checked(args, stream);
}

int eg2_hip_heads_norm_rope(const eg2_heads_norm_rope_args* args, void* stream) {
  return checked(args, stream);
}

int eg2_hip_window_attention(const eg2_window_attention_args* args, void* stream) {
  return checked(args, stream);
}

uint64_t eg2_hip_window_attention_workspace(const eg2_window_attention_args* args) {
  return args && valid_sizes(*args) ? eg2::block::window_attention_workspace(*args) : 0;
}

}  // extern "C"
