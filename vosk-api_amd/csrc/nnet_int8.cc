// The 8-bit form of a looped nnet3 plan (see nnet_int8.h).
#include "nnet_int8.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <limits>
#include <sstream>

#include "common.h"
#include "int8_ops.h"

namespace vamd {

float QuantizeRow(const float* x, int k, int8_t* codes) {
  float top = 0.0f;
  bool fine = true;
  for (int i = 0; i < k; i++) {
    fine = fine && std::isfinite(x[i]);
    top = std::max(top, std::fabs(x[i]));
  }
  const float s = top / 127.0f;
  for (int i = 0; i < k; i++) {
    const double q = fine && s > 0.0f ? std::nearbyint((double)x[i] / (double)s) : 0.0;  // halves to even
    codes[i] = (int8_t)std::min(127.0, std::max(-127.0, q));
  }
  return fine ? s : std::numeric_limits<float>::quiet_NaN();
}

namespace {

bool EvenlySpaced(const Op& op, int* step) {
  const std::vector<int>& p = op.pattern;
  if (p.empty()) return false;
  *step = p.size() > 1 ? p[1] - p[0] : 1;
  if (*step < 1) return false;
  for (size_t i = 1; i < p.size(); i++)
    if (p[i] - p[i - 1] != *step) return false;
  return true;
}

// The op's stages as the product's epilogue; false: they are something else.
bool TakeStages(const NnetPlan& p, const Op& op, Int8Plan::OpPlan* o) {
  int at = 0;  // bias, ReLU, scale + offset, bypass: each at most once, in this order
  for (const EpiStage& e : op.epi) {
    const int rank = e.kind == EpiStage::BIAS ? 1 : e.kind == EpiStage::RELU ? 2 : e.kind == EpiStage::ADD_NODE ? 4 : 3;
    if (rank <= at) return false;
    at = rank;
    if (e.kind == EpiStage::BIAS) {
      o->bias = e.vec0;
    } else if (e.kind == EpiStage::RELU) {
      o->relu = true;
    } else if (e.kind == EpiStage::MUL_ADD) {
      o->gain = p.vecs[e.vec0];
      o->shift = p.vecs[e.vec1];
    } else if (e.kind == EpiStage::SCALE) {
      o->gain.assign(op.N, e.c);
      o->shift.assign(op.N, 0.0f);
    } else {
      if (e.node == p.input_node || e.node == p.ivector_node) return false;
      o->res_node = e.node;
      o->res_src = e.src_col;
      o->res_scale = e.scaled ? e.c : 1.0f;
    }
  }
  return true;
}

}  // namespace

Int8Plan BuildInt8Plan(const NnetPlan& p) {
  Int8Plan r;
  r.ops.resize(p.ops.size());
  r.coded.assign(p.nodes.size(), 0);
  std::vector<int> producer(p.nodes.size(), -1);
  for (size_t i = 0; i < p.ops.size(); i++)
    if (p.ops[i].out_node >= 0) producer[p.ops[i].out_node] = (int)i;

  for (size_t i = 0; i < p.ops.size(); i++) {
    const Op& op = p.ops[i];
    int step, from;
    if (op.kind != Op::GEMM || op.segs.empty() || !EvenlySpaced(op, &step)) continue;
    const int node = op.segs[0].node;
    if (node == p.input_node || node == p.ivector_node || producer[node] < 0) continue;
    if (p.ops[producer[node]].kind != Op::GEMM || !EvenlySpaced(p.ops[producer[node]], &from)) continue;
    const int dim = p.nodes[node].dim;
    bool whole = (int)op.segs.size() + 2 <= kMaxTaps && dim <= kInt8MaxK;
    for (size_t j = 0; j < op.segs.size(); j++) {
      const ASegment& s = op.segs[j];
      whole = whole && s.node == node && s.dim == dim && s.src_col == 0 && s.col0 == (int)j * dim;
    }
    Int8Plan::OpPlan o;
    if (!whole || !TakeStages(p, op, &o)) continue;
    o.product = true;
    o.node = node;
    o.taps = (int)op.segs.size();
    o.k = Int8Padded(dim);
    o.w.assign((size_t)op.N * o.taps * o.k, 0);
    o.wscale.resize(op.N);
    std::vector<int8_t> row(op.K);
    const Matrix& w = p.mats[op.weight];
    for (int n = 0; n < op.N; n++) {
      o.wscale[n] = QuantizeRow(w.row(n), op.K, row.data());
      for (int j = 0; j < o.taps; j++)
        std::copy(row.begin() + j * dim, row.begin() + (j + 1) * dim, o.w.begin() + ((size_t)n * o.taps + j) * o.k);
    }
    r.ops[i] = std::move(o);
    r.coded[node] = 1;
    r.products++;
  }

  // columns of the maps: ops of the same number and spacing of rows share a
  // launch until its columns are full
  for (size_t i = 0; i < p.ops.size(); i++) {
    const Op& op = p.ops[i];
    Int8Plan::OpPlan& o = r.ops[i];
    o.quantize = op.out_node >= 0 && r.coded[op.out_node];
    if (!o.product && !o.quantize) continue;
    int step;
    EvenlySpaced(op, &step);
    std::vector<int> need;
    const int t0 = op.pattern[0];
    for (int j = 0; j < o.taps; j++) need.push_back(t0 + op.segs[j].offset);
    if (op.out_node >= 0) need.push_back(t0);
    if (o.res_node >= 0)
      for (const EpiStage& e : op.epi)
        if (e.kind == EpiStage::ADD_NODE) need.push_back(t0 + e.offset);
    for (size_t m = 0; m < r.maps.size() && o.map < 0; m++)
      if (r.maps[m].step == step && r.maps[m].rows == (int)op.pattern.size() &&
          r.maps[m].offsets.size() + need.size() <= (size_t)kMaxTaps)
        o.map = (int)m;
    if (o.map < 0) {
      o.map = (int)r.maps.size();
      r.maps.push_back({step, (int)op.pattern.size(), {}});
    }
    std::vector<int>& cols = r.maps[o.map].offsets;
    o.col = (int)cols.size();
    if (op.out_node >= 0) o.out_col = o.col + o.taps;
    if (o.res_node >= 0) o.res_col = o.col + o.taps + (op.out_node >= 0 ? 1 : 0);
    cols.insert(cols.end(), need.begin(), need.end());
  }
  for (const Int8Plan::Map& m : r.maps) {
    const auto mm = std::minmax_element(m.offsets.begin(), m.offsets.end());
    r.span = std::max(r.span, (m.rows - 1) * m.step + *mm.second - *mm.first + 1);
  }
  return r;
}

long long Int8Plan::MaxRingRows(const NnetPlan& p) const {
  long long rows = INT_MAX;
  auto mapped = [&](int node) {
    if (node >= 0) rows = std::min(rows, ((1ll << 31) - 1) / ((long long)sizeof(float) * p.nodes[node].dim));
  };
  for (size_t i = 0; i < ops.size(); i++) {
    if (!ops[i].product) continue;
    mapped(p.ops[i].out_node);
    mapped(ops[i].res_node);
  }
  return rows;
}

std::string Int8Plan::Describe(const NnetPlan& p) const {
  std::ostringstream os;
  for (size_t i = 0; i < ops.size(); i++) {
    const OpPlan& o = ops[i];
    if (!o.product && !o.quantize) continue;
    os << p.ops[i].name << ":";
    if (o.product) os << " product of " << p.nodes[o.node].name << " x " << o.taps;
    if (o.res_node >= 0) os << " + " << o.res_scale << " * " << p.nodes[o.res_node].name;
    if (o.quantize) os << " -> codes";
    os << " (map " << o.map << ")\n";
  }
  os << products << " products, " << maps.size() << " maps\n";
  return os.str();
}

}  // namespace vamd
