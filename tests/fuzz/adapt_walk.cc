// Speaker adaptation by distillation through the classes, as a program would do it: a teacher's largest logits (cu::RowTop),
// a shared hidden layer with the speakers' low-rank adapters (Adapters, AdapterRows), the loss towards the teacher mixed with
// hard labels (Distill), the way back through the output layer and the adapters' step.  Everything it starts from and every
// intermediate result goes to a dump; tests/test_gpu_adapt_walk.py does the same in 64 bits.
//
// usage: adapt_walk <seed> <steps> <dump-file> <adapters-file>
#include <cstdio>
#include <cstdlib>
#include <fstream>
#include <iostream>
#include <string>
#include <vector>

#include "base/kaldi-common.h"
#include "cudamatrix/cu-math.h"
#include "nnet/nnet-adapters.h"
#include "nnet/nnet-biasedlinearity.h"
#include "nnet/nnet-loss.h"

using namespace kaldi;

namespace {
struct Lcg {
  unsigned long long s;
  explicit Lcg(unsigned long long seed) : s(seed * 2862933555777941757ULL + 3037000493ULL) {}
  unsigned next() {
    s = s * 6364136223846793005ULL + 1442695040888963407ULL;
    return static_cast<unsigned>(s >> 33);
  }
  int below(int n) { return static_cast<int>(next() % static_cast<unsigned>(n)); }
  float sym() { return 2.0f * ((next() & 0xffffff) / 16777216.0f) - 1.0f; }
};

FILE *g_out = NULL;
void Dump(const char *name, const CuMatrix<BaseFloat> &m) {
  Matrix<BaseFloat> h;
  m.CopyToMat(&h);
  fprintf(g_out, "%s %d %d", name, h.NumRows(), h.NumCols());
  for (int32 r = 0; r < h.NumRows(); ++r)
    for (int32 c = 0; c < h.NumCols(); ++c) fprintf(g_out, " %.9g", h(r, c));
  fprintf(g_out, "\n");
}
void Dump(const char *name, const std::vector<float> &v) {
  fprintf(g_out, "%s 1 %d", name, static_cast<int>(v.size()));
  for (size_t i = 0; i < v.size(); ++i) fprintf(g_out, " %.9g", v[i]);
  fprintf(g_out, "\n");
}
void Dump(const char *name, const CuStlVector<int32> &d) {
  std::vector<int32> v;
  d.CopyToVec(&v);
  Dump(name, std::vector<float>(v.begin(), v.end()));
}
Matrix<BaseFloat> Random(Lcg *g, int32 rows, int32 cols, float scale) {
  Matrix<BaseFloat> m(rows, cols);
  for (int32 r = 0; r < rows; ++r)
    for (int32 c = 0; c < cols; ++c) m(r, c) = scale * g->sym();
  return m;
}
}  // namespace

int main(int argc, char **argv) {
  if (argc != 5) {
    fprintf(stderr, "usage: adapt_walk <seed> <steps> <dump-file> <adapters-file>\n");
    return 1;
  }
  try {
    CuDevice::Instantiate().SelectGpuId(-1);
    g_out = fopen(argv[3], "w");
    if (!g_out) KALDI_ERR << "cannot write " << argv[3];
    Lcg g(atoi(argv[1]));
    const int32 steps = atoi(argv[2]);
    const int32 rows = 20 + g.below(300), in = 10 + g.below(90), hid = 8 + g.below(120), out = 20 + g.below(400);
    const int32 num = 1 + g.below(9), k = 1 + g.below(12);

    BiasedLinearity layer1(in, hid, NULL), layer2(hid, out, NULL);
    CuMatrix<BaseFloat> x, teacher;
    CuVector<BaseFloat> b1, b2;
    Matrix<BaseFloat> w1 = Random(&g, hid, in, 0.5f), w2 = Random(&g, out, hid, 0.5f);
    layer1.SetLinearityWeight(w1, false);
    layer2.SetLinearityWeight(w2, false);
    Vector<BaseFloat> v1(hid), v2(out);
    for (int32 i = 0; i < hid; ++i) v1(i) = g.sym();
    for (int32 i = 0; i < out; ++i) v2(i) = g.sym();
    layer1.SetBiasWeight(v1);
    layer2.SetBiasWeight(v2);
    x.CopyFromMat(Random(&g, rows, in, 1.0f));
    teacher.CopyFromMat(Random(&g, rows, out, 4.0f));

    std::vector<int32> ranks, ids, labels;
    std::vector<BaseFloat> scale;
    int32 total = 0;
    for (int32 i = 0; i < num; ++i) {
      ranks.push_back(g.below(7));
      total += ranks.back();
      scale.push_back(0.5f + 0.5f * (g.sym() + 1.0f));
    }
    for (int32 r = 0; r < rows; ++r) {
      ids.push_back(g.below(num + 1) - 1);
      labels.push_back(g.below(out));
    }
    CuVector<BaseFloat> weight;
    Vector<BaseFloat> hw(rows);
    for (int32 r = 0; r < rows; ++r) hw(r) = g.below(10) ? 1.0f + 0.5f * g.sym() : 0.0f;
    weight.CopyFromVec(hw);
    CuStlVector<int32> label;
    label.CopyFromVec(labels);

    Adapters adapters;
    adapters.Init(in, hid, ranks, scale);
    if (total > 0) {
      adapters.SetDown(Random(&g, total, in, 0.4f));
      adapters.SetUp(Random(&g, total, hid, 0.4f));
    }
    AdapterRows who;
    who.Set(ids, num, g.below(2) == 1);

    Dump("w1", layer1.GetLinearityWeight());
    Dump("w2", layer2.GetLinearityWeight());
    std::vector<float> tmp;
    for (int32 i = 0; i < hid; ++i) tmp.push_back(v1(i));
    Dump("b1", tmp);
    tmp.clear();
    for (int32 i = 0; i < out; ++i) tmp.push_back(v2(i));
    Dump("b2", tmp);
    Dump("x", x);
    Dump("teacher", teacher);
    Dump("ranks", std::vector<float>(ranks.begin(), ranks.end()));
    Dump("scale", std::vector<float>(scale.begin(), scale.end()));
    Dump("ids", std::vector<float>(ids.begin(), ids.end()));
    Dump("labels", std::vector<float>(labels.begin(), labels.end()));
    tmp.clear();
    for (int32 r = 0; r < rows; ++r) tmp.push_back(hw(r));
    Dump("weight", tmp);
    Dump("down", adapters.Down());
    Dump("up", adapters.Up());

    CuStlVector<int32> id;
    CuMatrix<BaseFloat> val;
    CuVector<BaseFloat> lse;
    cu::RowTop(teacher, k, &id, &val, &lse);
    Dump("id", id);
    Dump("val", val);

    Distill loss(2.0, 0.25);
    CuMatrix<BaseFloat> h, z, diff, err_h, err_x;
    for (int32 s = 0; s < steps; ++s) {
      adapters.Propagate(&layer1, x, who, KH_ACT_SIGMOID, &h);
      layer2.PropagateFused(h, KH_ACT_NONE, &z);
      loss.Eval(z, id, val, &label, &weight, &diff);
      layer2.BackpropagateFused(diff, h, &err_h);
      adapters.Backpropagate(&layer1, x, err_h, who, NULL, &err_x);
      Dump("h", h);
      Dump("diff", diff);
      Dump("err_x", err_x);
      if (total > 0) {
        Dump("down_grad", adapters.DownGradient());
        Dump("up_grad", adapters.UpGradient());
      }
      adapters.Update(0.01f);
    }
    int64 frames;
    double sum;
    loss.GetStats(&frames, &sum);
    fprintf(g_out, "loss 1 2 %.17g %lld\n", sum, static_cast<long long>(frames));
    Dump("down_end", adapters.Down());
    Dump("up_end", adapters.Up());
    std::cout << loss.Report() << std::endl;

    // out to a file and back, both ways
    for (int binary = 0; binary < 2; ++binary) {
      {
        std::ofstream os(argv[4], std::ios::binary);
        adapters.Write(os, binary != 0);
      }
      std::ifstream is(argv[4], std::ios::binary);
      Adapters again;
      again.Read(is, binary != 0);
      Dump(binary ? "down_binary" : "down_text", again.Down());
      Dump(binary ? "up_binary" : "up_text", again.Up());
      CuMatrix<BaseFloat> h2;
      again.Propagate(&layer1, x, who, KH_ACT_SIGMOID, &h2);
      adapters.Propagate(&layer1, x, who, KH_ACT_SIGMOID, &h);
      Dump(binary ? "h_binary" : "h_text", h2);
      Dump("h_end", h);
    }
    fclose(g_out);
    return 0;
  } catch (const std::exception &e) {
    std::cerr << e.what();
    return 255;
  }
}
