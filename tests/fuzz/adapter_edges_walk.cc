// The adapter classes where a call goes wrong or has nothing to do; tests/test_adapter_classes.py and
// tests/test_gpu_adapter_classes.py look at what is printed.
//
// usage: adapter_edges_walk read <adapters-file>    a file that is refused, into empty adapters (no device is needed)
//        adapter_edges_walk reread <adapters-file>  the same into adapters that are in use
//        adapter_edges_walk stale <adapters-file>   a good file into adapters that hold a forward pass and gradients
//        adapter_edges_walk empty                   a bunch without rows
//        adapter_edges_walk inplace                 outputs that are inputs, of the adapters, RowTop and Distill
#include <cstdio>
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

// true if the file was refused
bool Refused(Adapters *adapters, const char *file) {
  std::ifstream is(file, std::ios::binary);
  if (!is) {
    fprintf(stderr, "cannot read %s\n", file);
    exit(1);
  }
  try {
    adapters->Read(is, false);
  } catch (const std::exception &e) {
    std::cerr << e.what();
    return true;
  }
  return false;
}

void Fill(Matrix<BaseFloat> *m, float scale) {
  for (int32 r = 0; r < m->NumRows(); ++r)
    for (int32 c = 0; c < m->NumCols(); ++c) (*m)(r, c) = scale * static_cast<float>((7 * r + 3 * c) % 11 - 5);
}

// a layer, the adapters of some speakers and a bunch of rows
struct Bench {
  static const int32 kRows = 37, kIn = 12, kOut = 9;
  BiasedLinearity layer;
  CuMatrix<BaseFloat> x, err;
  Adapters adapters;
  AdapterRows who;
  int32 num;
  Bench() : layer(kIn, kOut, NULL), num(3) {
    Matrix<BaseFloat> w(kOut, kIn), in(kRows, kIn), e(kRows, kOut), down(6, kIn), up(6, kOut);
    Vector<BaseFloat> b(kOut);
    for (int32 i = 0; i < kOut; ++i) b(i) = 0.1f * i;
    Fill(&w, 0.05f);
    Fill(&in, 0.2f);
    Fill(&e, 0.1f);
    Fill(&down, 0.1f);
    Fill(&up, 0.1f);
    layer.SetLinearityWeight(w, false);
    layer.SetBiasWeight(b);
    x.CopyFromMat(in);
    err.CopyFromMat(e);
    adapters.Init(kIn, kOut, std::vector<int32>({1, 2, 3}), std::vector<BaseFloat>({1.0f, 0.5f, 2.0f}));
    adapters.SetDown(down);
    adapters.SetUp(up);
    std::vector<int32> ids;
    for (int32 r = 0; r < kRows; ++r) ids.push_back(r % (num + 1) - 1);
    who.Set(ids, num);
  }
};

std::vector<float> Values(const CuMatrix<BaseFloat> &m) {
  Matrix<BaseFloat> h;
  m.CopyToMat(&h);
  std::vector<float> v;
  for (int32 r = 0; r < h.NumRows(); ++r)
    for (int32 c = 0; c < h.NumCols(); ++c) v.push_back(h(r, c));
  return v;
}

int Read(const char *file) {
  Adapters a;
  const bool refused = Refused(&a, file);
  printf("refused %d adapters %d %d -> %d\n", refused, a.NumAdapters(), a.InputDim(), a.OutputDim());
  return 0;
}

int Reread(const char *file) {
  Bench s;
  CuMatrix<BaseFloat> before, after;
  s.adapters.Propagate(&s.layer, s.x, s.who, KH_ACT_SIGMOID, &before);
  const bool refused = Refused(&s.adapters, file);
  printf("refused %d adapters %d %d -> %d\n", refused, s.adapters.NumAdapters(), s.adapters.InputDim(), s.adapters.OutputDim());
  fflush(stdout);
  s.adapters.Propagate(&s.layer, s.x, s.who, KH_ACT_SIGMOID, &after);
  printf("same %d\n", Values(before) == Values(after));
  return 0;
}

template <class F>
bool Throws(F f) {
  try {
    f();
  } catch (const std::exception &e) {
    std::cerr << e.what();
    return true;
  }
  return false;
}

int Stale(const char *file) {
  Bench s;
  CuMatrix<BaseFloat> out;
  s.adapters.Propagate(&s.layer, s.x, s.who, KH_ACT_SIGMOID, &out);
  s.adapters.Backpropagate(&s.layer, s.x, s.err, s.who, NULL, NULL);
  {
    std::ofstream os(file, std::ios::binary);
    s.adapters.Write(os, true);
  }
  std::ifstream is(file, std::ios::binary), is2(file, std::ios::binary);
  Adapters fresh;
  fresh.Read(is, true);
  s.adapters.Read(is2, true);
  const std::vector<float> down = Values(s.adapters.Down()), up = Values(s.adapters.Up());
  printf("update refused %d\n", Throws([&] { s.adapters.Update(0.1f); }));
  printf("weights same %d\n", down == Values(s.adapters.Down()) && up == Values(s.adapters.Up()));
  printf("backpropagate refused %d\n", Throws([&] { s.adapters.Backpropagate(&s.layer, s.x, s.err, s.who, NULL, NULL); }));
  Adapters *both[2] = {&s.adapters, &fresh};
  for (int i = 0; i < 2; ++i) {
    both[i]->Propagate(&s.layer, s.x, s.who, KH_ACT_SIGMOID, &out);
    both[i]->Backpropagate(&s.layer, s.x, s.err, s.who, NULL, NULL);
    both[i]->Update(0.1f);
  }
  printf("as fresh ones %d\n", Values(s.adapters.Down()) == Values(fresh.Down()) && Values(s.adapters.Up()) == Values(fresh.Up()) &&
                                    Values(fresh.Up()) != up);
  return 0;
}

bool AllZero(const CuMatrix<BaseFloat> &m, int32 rows, int32 cols) {
  const std::vector<float> v = Values(m);
  for (size_t i = 0; i < v.size(); ++i)
    if (v[i] != 0.0f) return false;
  return m.NumRows() == rows && m.NumCols() == cols;
}

int Empty() {
  Bench s;
  CuMatrix<BaseFloat> out, below, nothing;
  AdapterRows none;
  none.Set(std::vector<int32>(), s.num);
  for (int turn = 0; turn < 2; ++turn) {  // behind nothing, and behind a bunch with rows
    s.adapters.Propagate(&s.layer, nothing, none, KH_ACT_SIGMOID, &out);
    s.adapters.Backpropagate(&s.layer, nothing, nothing, none, &nothing, &below);
    printf("out %d below %d gradients zero %d\n", out.NumRows(), below.NumRows(),
           AllZero(s.adapters.DownGradient(), 6, s.kIn) && AllZero(s.adapters.UpGradient(), 6, s.kOut));
    s.adapters.Update(1.0f);
    s.adapters.Propagate(&s.layer, s.x, s.who, KH_ACT_SIGMOID, &out);
    s.adapters.Backpropagate(&s.layer, s.x, s.err, s.who, &s.x, &below);
    printf("out %d below %d gradients zero %d\n", out.NumRows(), below.NumRows(),
           AllZero(s.adapters.DownGradient(), 6, s.kIn) && AllZero(s.adapters.UpGradient(), 6, s.kOut));
  }
  return 0;
}

int InPlace() {
  Bench s;
  CuMatrix<BaseFloat> out, y, val;
  s.adapters.Propagate(&s.layer, s.x, s.who, KH_ACT_SIGMOID, &out);
  const std::vector<float> x = Values(s.x), err = Values(s.err), o = Values(out);
  y.CopyFromMat(s.x);
  printf("propagate refused %d\n", Throws([&] { s.adapters.Propagate(&s.layer, s.x, s.who, KH_ACT_SIGMOID, &s.x); }));
  printf("backpropagate refused %d %d %d\n", Throws([&] { s.adapters.Backpropagate(&s.layer, s.x, s.err, s.who, &y, &s.x); }),
         Throws([&] { s.adapters.Backpropagate(&s.layer, s.x, s.err, s.who, &y, &s.err); }),
         Throws([&] { s.adapters.Backpropagate(&s.layer, s.x, s.err, s.who, &y, &y); }));
  CuStlVector<int32> id;
  printf("row top refused %d\n", Throws([&] { cu::RowTop(out, 4, &id, &out, static_cast<CuVector<BaseFloat> *>(NULL)); }));
  cu::RowTop(out, 4, &id, &val, static_cast<CuVector<BaseFloat> *>(NULL));
  const std::vector<float> v = Values(val);
  Distill loss(2.0, 0.0);
  printf("distill refused %d\n", Throws([&] { loss.Eval(out, id, val, NULL, NULL, &val); }));
  printf("inputs same %d\n", Values(s.x) == x && Values(s.err) == err && Values(out) == o && Values(y) == x && Values(val) == v);
  loss.Eval(out, id, val, NULL, NULL, &out);  // (the gradient may take the logits' place)
  printf("in place %d\n", Values(out) != o && out.NumRows() == s.kRows);
  return 0;
}

}  // namespace

int main(int argc, char **argv) {
  const std::string what = argc > 1 ? argv[1] : "";
  try {
    if (what == "read" && argc == 3) return Read(argv[2]);
    CuDevice::Instantiate().SelectGpuId(-1);
    if (what == "reread" && argc == 3) return Reread(argv[2]);
    if (what == "inplace" && argc == 2) return InPlace();
    if (what == "empty" && argc == 2) return Empty();
    if (what == "stale" && argc == 3) return Stale(argv[2]);
    fprintf(stderr, "usage: adapter_edges_walk read|reread|stale <adapters-file> | empty | inplace\n");
    return 1;
  } catch (const std::exception &e) {
    std::cerr << e.what();
    return 255;
  }
}
