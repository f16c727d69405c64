// Low-rank adapters of many speakers beside one shared <biasedlinearity> layer:
//   out = act( in * W^T + b + s_g (in * down_g^T) * up_g ),   g = the speaker of the row.
// No counterpart in the reference.  W and b are the layer's and stay as they are; the adapters of a layer lie below each
// other in two matrices (down: input_dim columns, up: output_dim columns), so that one launch serves all speakers of a
// bunch.
#ifndef KALDI_AMD_NNET_NNET_ADAPTERS_H_
#define KALDI_AMD_NNET_NNET_ADAPTERS_H_
#include <limits>
#include <vector>

#include "base/io-funcs.h"
#include "cudamatrix/cu-math.h"
#include "cudamatrix/cu-stlvector.h"
#include "nnet/nnet-biasedlinearity.h"

namespace kaldi {

/// Which adapter each row of a bunch takes (anything outside [0, num) = none), and the rows grouped by adapter.  One
/// serves every adapted layer, forward and backward.
class AdapterRows {
 public:
  /// `grouped`: rows of one speaker lie together already (utterances, single frames), so tiles are taken in row order; the
  /// grouping is made all the same, the gradients need it.
  void Set(const std::vector<int32> &row_adapter, int32 num, bool grouped = false) {
    row_adapter_.CopyFromVec(row_adapter);
    Plan(num, grouped);
  }
  void Set(const CuStlVector<int32> &row_adapter, int32 num, bool grouped = false) {
    row_adapter_.CopyFromCuVec(row_adapter, 0, row_adapter.Dim());
    Plan(num, grouped);
  }
  int32 NumRows() const { return static_cast<int32>(row_adapter_.Dim()); }
  int32 NumAdapters() const { return num_; }
  const int32 *RowAdapter() const { return row_adapter_.Data(); }
  const int32 *TileOrder() const { return grouped_ ? NULL : order_.Data(); }
  const CuStlVector<int32> &Order() const { return order_; }
  const CuStlVector<int32> &RowBegin() const { return row_begin_; }

 private:
  void Plan(int32 num, bool grouped) {
    KALDI_ASSERT(num >= 0);
    num_ = num;
    grouped_ = grouped;
    order_.Resize(row_adapter_.Dim());
    row_begin_.Resize(num + 1);
    CU_SAFE_CALL(hipI32_adapter_plan(CuDevice::Instantiate().Stream(), row_adapter_.Data(), NumRows(), num, order_.Data(),
                                     row_begin_.Data()));
  }
  CuStlVector<int32> row_adapter_, order_, row_begin_;
  int32 num_ = 0;
  bool grouped_ = false;
};

class Adapters {
 public:
  Adapters() {}

  /// Adapters of the given ranks (each 0 .. KH_MAX_ADAPTER_RANK) for a layer input_dim -> output_dim, all weights 0.  What is
  /// refused leaves the adapters as they were; where the device has no memory for the new ones, there are none afterwards.
  void Init(int32 input_dim, int32 output_dim, const std::vector<int32> &ranks, const std::vector<BaseFloat> &scale) {
    KALDI_ASSERT(input_dim > 0 && output_dim > 0 && ranks.size() == scale.size());
    std::vector<int32> begin(1, 0);
    int32 max_rank = 1;
    int64 rows = 0;
    for (size_t g = 0; g < ranks.size(); ++g) {
      if (ranks[g] < 0 || ranks[g] > KH_MAX_ADAPTER_RANK)
        KALDI_ERR << "Adapter " << g << " of rank " << ranks[g] << ": 0 to " << KH_MAX_ADAPTER_RANK << " are supported";
      rows += ranks[g];
      if (rows > std::numeric_limits<int32>::max()) KALDI_ERR << "Adapters of more than 2^31 - 1 rows together";
      begin.push_back(static_cast<int32>(rows));
      if (ranks[g] > max_rank) max_rank = ranks[g];
    }
    // none, until everything is there: the number of adapters is what the kernels read `begin` and `scale` by
    ranks_.clear();
    input_dim_ = output_dim_ = 0;
    t_.Resize(0, 0);  // (what a forward and a backward pass left is of the adapters before)
    u_.Resize(0, 0);
    down_grad_.Resize(0, 0);
    up_grad_.Resize(0, 0);
    begin_.CopyFromVec(begin);
    Vector<BaseFloat> s(scale.size());
    for (size_t g = 0; g < scale.size(); ++g) s(g) = scale[g];
    scale_.CopyFromVec(s);
    down_.Resize(begin.back(), input_dim);
    up_.Resize(begin.back(), output_dim);
    down_.SetZero();
    up_.SetZero();
    max_rank_ = max_rank;
    input_dim_ = input_dim;
    output_dim_ = output_dim;
    ranks_ = ranks;
  }

  int32 NumAdapters() const { return static_cast<int32>(ranks_.size()); }
  int32 InputDim() const { return input_dim_; }
  int32 OutputDim() const { return output_dim_; }
  /// the stacks, adapter g at the rows behind the ranks of 0 .. g-1
  const CuMatrix<BaseFloat> &Down() const { return down_; }
  const CuMatrix<BaseFloat> &Up() const { return up_; }
  void SetDown(const Matrix<BaseFloat> &m) {
    KALDI_ASSERT(m.NumRows() == down_.NumRows() && m.NumCols() == down_.NumCols());
    down_.CopyFromMat(m);
  }
  void SetUp(const Matrix<BaseFloat> &m) {
    KALDI_ASSERT(m.NumRows() == up_.NumRows() && m.NumCols() == up_.NumCols());
    up_.CopyFromMat(m);
  }
  /// of the last Backpropagate
  const CuMatrix<BaseFloat> &DownGradient() const { return down_grad_; }
  const CuMatrix<BaseFloat> &UpGradient() const { return up_grad_; }

  /// out = act( layer(in) + adapters ), act = KH_ACT_NONE | KH_ACT_SIGMOID | KH_ACT_SOFTMAX
  void Propagate(BiasedLinearity *layer, const CuMatrix<BaseFloat> &in, const AdapterRows &rows, int act,
                 CuMatrix<BaseFloat> *out) {
    CuProfileScope p("Adapters::Propagate");
    Check(layer, in, rows);
    if (out == &in) KALDI_ERR << "Adapters: the output is the input";  // (it would be resized, and with that lost)
    if (out->NumRows() != in.NumRows() || out->NumCols() != output_dim_) out->Resize(in.NumRows(), output_dim_);
    t_.Resize(in.NumRows(), max_rank_);
    const khAdapters ad = Describe();
    const CuMatrix<BaseFloat> &W = layer->GetLinearityWeight();
    CU_SAFE_CALL(hipF_adapter_forward(S(), act, in.NumRows(), output_dim_, input_dim_, in.Data(), in.Stride(), W.Data(),
                                      W.Stride(), layer->GetBiasWeight().Data(), &ad, rows.RowAdapter(), rows.TileOrder(),
                                      t_.Data(), t_.Stride(), out->Data(), out->Stride()));
  }

  /// Behind Propagate of the same rows: the gradients of the stacks from the error at the layer's output (before its
  /// activation), and, unless out_err is NULL, the error of the layer below, times y (1 - y) of its sigmoid if y is given.
  void Backpropagate(BiasedLinearity *layer, const CuMatrix<BaseFloat> &in, const CuMatrix<BaseFloat> &in_err,
                     const AdapterRows &rows, const CuMatrix<BaseFloat> *y, CuMatrix<BaseFloat> *out_err) {
    CuProfileScope p("Adapters::Backpropagate");
    Check(layer, in, rows);
    KALDI_ASSERT(in_err.NumRows() == in.NumRows() && (in.NumRows() == 0 || in_err.NumCols() == output_dim_));
    if (t_.NumRows() != in.NumRows() || (in.NumRows() > 0 && t_.NumCols() != max_rank_))
      KALDI_ERR << "Adapters: no forward pass of these " << in.NumRows() << " rows";
    KALDI_ASSERT(y == NULL || (y->NumRows() == in.NumRows() && (in.NumRows() == 0 || y->NumCols() == input_dim_)));
    if (out_err && (out_err == &in || out_err == &in_err || out_err == y))
      KALDI_ERR << "Adapters: the error of the layer below is an input";
    if (out_err && (out_err->NumRows() != in.NumRows() || out_err->NumCols() != input_dim_))
      out_err->Resize(in.NumRows(), input_dim_);
    u_.Resize(in.NumRows(), max_rank_);
    down_grad_.Resize(down_.NumRows(), input_dim_);
    up_grad_.Resize(up_.NumRows(), output_dim_);
    const khAdapters ad = Describe();
    const CuMatrix<BaseFloat> &W = layer->GetLinearityWeight();
    CU_SAFE_CALL(hipF_adapter_backward(
        S(), in.NumRows(), output_dim_, input_dim_, in_err.Data(), in_err.Stride(), in.Data(), in.Stride(), W.Data(), W.Stride(),
        &ad, rows.RowAdapter(), rows.Order().Data(), rows.RowBegin().Data(), t_.Data(), t_.Stride(), u_.Data(), u_.Stride(),
        y ? y->Data() : NULL, y ? y->Stride() : 0, out_err ? out_err->Data() : NULL, out_err ? out_err->Stride() : 0,
        down_grad_.Data(), down_grad_.Stride(), up_grad_.Data(), up_grad_.Stride()));
  }

  /// a step against the gradients of the last Backpropagate; refused where Init or Read came behind it
  void Update(BaseFloat learn_rate) {
    CuProfileScope p("Adapters::Update");
    if (down_grad_.NumRows() != down_.NumRows() || up_grad_.NumRows() != up_.NumRows())
      KALDI_ERR << "Adapters: no gradients of these adapters";
    down_.AddMat(-learn_rate, down_grad_);
    up_.AddMat(-learn_rate, up_grad_);
  }

  void Write(std::ostream &os, bool binary) const {
    WriteToken(os, binary, "<adapters>");
    WriteBasicType(os, binary, output_dim_);
    WriteBasicType(os, binary, input_dim_);
    WriteIntegerVector(os, binary, ranks_);
    scale_.Write(os, binary);
    down_.Write(os, binary);
    up_.Write(os, binary);
  }
  void Read(std::istream &is, bool binary) {
    ExpectToken(is, binary, "<adapters>");
    int32 output_dim, input_dim;
    std::vector<int32> ranks;
    ReadBasicType(is, binary, &output_dim);
    ReadBasicType(is, binary, &input_dim);
    ReadIntegerVector(is, binary, &ranks);
    Vector<BaseFloat> scale;
    Matrix<BaseFloat> down, up;
    scale.Read(is, binary);
    down.Read(is, binary);
    up.Read(is, binary);
    if (output_dim <= 0 || input_dim <= 0 || static_cast<size_t>(scale.Dim()) != ranks.size())
      KALDI_ERR << "Adapters: " << ranks.size() << " ranks, " << scale.Dim() << " scales, " << input_dim << " -> " << output_dim;
    std::vector<BaseFloat> s(ranks.size());
    int64 rows = 0;
    for (size_t g = 0; g < s.size(); ++g) {
      s[g] = scale(g);
      rows += ranks[g];
    }
    if (down.NumRows() != rows || up.NumRows() != rows ||
        (rows > 0 && (down.NumCols() != input_dim || up.NumCols() != output_dim)))
      KALDI_ERR << "Adapters: stacks of " << down.NumRows() << " and " << up.NumRows() << " rows, the ranks add up to " << rows;
    Init(input_dim, output_dim, ranks, s);
    if (down.NumRows() > 0) {
      SetDown(down);
      SetUp(up);
    }
  }

 private:
  static khStream_t S() { return CuDevice::Instantiate().Stream(); }
  khAdapters Describe() const {
    khAdapters ad = {NumAdapters(), max_rank_, down_.NumRows(), begin_.Data(), scale_.Data(),
                     down_.Data(), down_.NumRows() > 0 ? down_.Stride() : input_dim_,
                     up_.Data(), up_.NumRows() > 0 ? up_.Stride() : output_dim_};
    return ad;
  }
  void Check(BiasedLinearity *layer, const CuMatrix<BaseFloat> &in, const AdapterRows &rows) const {
    // (a matrix without rows has no columns either)
    if (layer->InputDim() != input_dim_ || layer->OutputDim() != output_dim_ ||
        (in.NumRows() > 0 && in.NumCols() != input_dim_))
      KALDI_ERR << "Nonmatching dims, adapters:" << input_dim_ << "->" << output_dim_ << " layer:" << layer->InputDim() << "->"
                << layer->OutputDim() << " data:" << in.NumCols();
    KALDI_ASSERT(rows.NumRows() == in.NumRows() && rows.NumAdapters() == NumAdapters());
  }

  int32 input_dim_ = 0, output_dim_ = 0, max_rank_ = 1;
  std::vector<int32> ranks_;
  CuStlVector<int32> begin_;
  CuVector<BaseFloat> scale_;
  CuMatrix<BaseFloat> down_, up_, down_grad_, up_grad_;
  CuMatrix<BaseFloat> t_, u_;  // narrow products of the last Propagate / Backpropagate
};

}  // namespace kaldi
#endif
