// The optimizer operators' host code over a model of the HIP runtime, on the
// CPU: which launches a call makes, with which grids and tables, and that a
// refused call makes none.  The kernels themselves do not run.
//
// Usage: step_launches SCENARIO; prints "ok" and exits 0, or says what differs.
#include "../../suika_amd/csrc/optim.hip"

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>

namespace sr_internal {

char message[512];

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(message, sizeof message, fmt, ap);
  va_end(ap);
  return code;
}

int dtype_size(int32_t dt) { return dt == SR_DT_F32 ? 4 : dt == SR_DT_BF16 || dt == SR_DT_F16 ? 2 : 8; }

}  // namespace sr_internal

namespace model {

[[noreturn]] void die(const char* what) {
  std::printf("FAILED: %s (%s)\n", what, sr_internal::message);
  std::exit(1);
}

struct Launch {
  const void* fn;
  uint64_t blocks, threads;         // of the grid, of a block
  std::vector<unsigned char> table; // the last argument's bytes, where it is a table of the AdamW kernels
};
std::vector<Launch> launches;
bool capturing = false;

const void* const kCopies[] = {reinterpret_cast<const void*>(adamw_kernel<float, float, float, bf16>),
                               reinterpret_cast<const void*>(adamw_kernel<float, float, bf16, bf16>)};
const void* const kAlone[] = {reinterpret_cast<const void*>(adamw_kernel<float, float, float, NoCopy>),
                              reinterpret_cast<const void*>(adamw_kernel<float, float, bf16, NoCopy>),
                              reinterpret_cast<const void*>(adamw_kernel<bf16, bf16, bf16, NoCopy>)};

template <typename T>
std::vector<unsigned char> bytes_at(void* p) {
  std::vector<unsigned char> b(sizeof(T));
  std::memcpy(b.data(), p, sizeof(T));
  return b;
}

}  // namespace model

extern "C" {

hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "error of the model"; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* c) {
  return *c = model::capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone, hipSuccess;
}
hipError_t hipLaunchKernel(const void* fn, dim3 grid, dim3 block, void** args, size_t, hipStream_t) {
  model::Launch l{fn, uint64_t(grid.x), uint64_t(block.x), {}};
  for (const void* f : model::kCopies)
    if (f == fn) l.table = model::bytes_at<AdamTable<true>>(args[1]);
  for (const void* f : model::kAlone)
    if (f == fn) l.table = model::bytes_at<AdamTable<false>>(args[1]);
  model::launches.push_back(l);
  return hipSuccess;
}

static struct {
  dim3 grid, block;
  size_t shmem;
  hipStream_t stream;
} g_call;
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t m, hipStream_t s) {
  return g_call = {g, b, m, s}, hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* m, hipStream_t* s) {
  return *g = g_call.grid, *b = g_call.block, *m = g_call.shmem, *s = g_call.stream, hipSuccess;
}
void** __hipRegisterFatBinary(const void*) { return nullptr; }
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*, void*, int*) {}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
void __hipUnregisterFatBinary(void**) {}

}  // extern "C"

// ------------------------------------------------------------------ scenarios

namespace {

using model::die;
using model::launches;

constexpr uint64_t kBase = uint64_t(1) << 40;       // addresses that nothing reads
void* at(uint64_t offset) { return reinterpret_cast<void*>(kBase + offset); }

const sr_adamw_options kOptions = {1e-3, 0.9, 0.99, 1e-8, 0.1, 1, 1.0};

// The sum, the norm and a workspace, below all arrays.
const uint64_t kSum = -(uint64_t(1) << 21) + 64, kNorm = kSum + 32, kWork = kSum + 64;
sr_norm own_norm() {
  return {nullptr, static_cast<double*>(at(kSum)), at(kWork), 1 << 20, static_cast<float*>(at(kNorm))};
}

void expect(int rc, int want, size_t n, const char* what) {
  if (rc != want || launches.size() != n) {
    std::printf("status %d, %zu launches; wanted %d and %zu\n", rc, launches.size(), want, n);
    die(what);
  }
  launches.clear();
}

// Calls that form the sum themselves refuse before it is launched.
void refusals() {
  const uint64_t M = 1 << 24;
  const sr_norm norm = own_norm();
  const sr_array good[2] = {{at(M), 100000, SR_DT_F32, 0}, {at(2 * M), 8, SR_DT_BF16, 0}};
  const sr_array twice[2] = {good[0], good[0]};
  expect(sr_clip_norm(good, nullptr, 2, 1.0f, &norm, nullptr), SR_OK, 5, "clip");
  expect(sr_clip_norm(twice, nullptr, 2, 1.0f, &norm, nullptr), SR_EOVERLAP, 0, "clip: listed twice");
  expect(sr_clip_norm(good, nullptr, 2, -1.0f, &norm, nullptr), SR_EINVAL, 0, "clip: max_norm");
  expect(sr_clip_norm(good, nullptr, 2, 1.0f, nullptr, nullptr), SR_EINVAL, 0, "clip: no norm");
  sr_norm small = norm;
  small.workspace_bytes = 8;
  expect(sr_clip_norm(good, nullptr, 2, 1.0f, &small, nullptr), SR_EINVAL, 0, "clip: workspace");
  small = norm;
  small.sum = nullptr;
  expect(sr_clip_norm(good, nullptr, 2, 1.0f, &small, nullptr), SR_EINVAL, 0, "clip: no place for the sum");

  sr_adamw_tensor t{at(M), at(2 * M), at(3 * M), nullptr, at(4 * M), 100000, SR_DT_F32, SR_DT_F32, SR_DT_F32, 0};
  expect(sr_adamw_norm(&t, nullptr, 1, &kOptions, &norm, nullptr), SR_OK, 3, "adamw");
  expect(sr_adamw_norm(&t, nullptr, 1, &kOptions, nullptr, nullptr), SR_OK, 1, "adamw without clipping");
  sr_norm given = {norm.sum, nullptr, nullptr, 0, norm.norm};
  expect(sr_adamw_norm(&t, nullptr, 1, &kOptions, &given, nullptr), SR_OK, 2, "adamw by a given sum");
  given.norm = nullptr;
  expect(sr_adamw_norm(&t, nullptr, 1, &kOptions, &given, nullptr), SR_OK, 1, "adamw by a given sum alone");
  expect(sr_adamw_norm(&t, nullptr, 1, &kOptions, &small, nullptr), SR_EINVAL, 0, "adamw: no place for the sum");
  sr_adamw_options o = kOptions;
  o.lr = -1;
  expect(sr_adamw_norm(&t, nullptr, 1, &o, &norm, nullptr), SR_EINVAL, 0, "adamw: lr");
  o = kOptions;
  o.max_norm = -1;
  expect(sr_adamw_norm(&t, nullptr, 1, &o, &norm, nullptr), SR_EINVAL, 0, "adamw: max_norm");
  o.max_norm = 1;
  const sr_adamw_tensor both[2] = {t, t};
  expect(sr_adamw_norm(both, nullptr, 2, &o, &norm, nullptr), SR_EOVERLAP, 0, "adamw: listed twice");
  model::capturing = true;
  expect(sr_adamw_norm(&t, nullptr, 1, &o, &norm, nullptr), SR_EINVAL, 0, "adamw: captured");
  expect(sr_clip_norm(good, nullptr, 2, 1.0f, &norm, nullptr), SR_OK, 5, "clip: captured");
}

template <bool COPY>
const AdamTable<COPY>& table(size_t i) { return *reinterpret_cast<const AdamTable<COPY>*>(launches[i].table.data()); }

bool near(float got, double want) { return std::fabs(got - want) <= std::fabs(want) * 1e-7; }

// Tensors of other update numbers get their own bias corrections: launches by
// number, within one by type.
void steps() {
  const uint64_t M = 1 << 24;
  std::vector<sr_adamw_tensor> t;
  const int64_t numbers[6] = {7, 1, 7, 1000, 1, 7};
  for (int i = 0; i < 6; ++i) {
    const uint64_t b = uint64_t(i + 1) * M;
    t.push_back({at(b), at(b + 65536), at(b + 131072), i == 2 ? at(b + 196608) : nullptr, at(b + 262144), uint64_t(100 + i),
                 SR_DT_F32, SR_DT_F32, SR_DT_F32, 0});
  }
  if (sr_adamw_norm(t.data(), numbers, 6, &kOptions, nullptr, nullptr) != SR_OK) die("steps");
  // 1: two tensors; 7: one with a copy, two without; 1000: one
  const struct { int64_t step; std::vector<int> tensors; } want[4] = {{1, {1, 4}}, {7, {2}}, {7, {0, 5}}, {1000, {3}}};
  if (launches.size() != 4) die("launches by number and type");
  for (int k = 0; k < 4; ++k) {
    const double c1 = 1 - std::pow(0.9, double(want[k].step)), c2 = 1 - std::pow(0.99, double(want[k].step));
    const auto check = [&](const auto& tab) {
      if (!near(tab.step_size, 1e-3 / c1) || !near(tab.root_scale, 1 / std::sqrt(c2))) die("bias corrections");
      if (tab.at.count != want[k].tensors.size()) die("tensors of a launch");
      for (size_t j = 0; j < want[k].tensors.size(); ++j) {
        const sr_adamw_tensor& x = t[size_t(want[k].tensors[j])];
        if (tab.entry[j].weight != reinterpret_cast<uint64_t>(x.weight) || tab.tail[j] != x.n) die("another tensor");
      }
    };
    if (k == 1) check(table<true>(1));
    else check(table<false>(size_t(k)));
  }
  launches.clear();
  const int64_t same[6] = {7, 7, 7, 7, 7, 7};
  expect(sr_adamw_norm(t.data(), same, 6, &kOptions, nullptr, nullptr), SR_OK, 2, "one number");
  const int64_t none[6] = {7, 7, 0, 7, 7, 7};
  expect(sr_adamw_norm(t.data(), none, 6, &kOptions, nullptr, nullptr), SR_EINVAL, 0, "a number below 1");
  sr_adamw_options o = kOptions;
  o.step = 0;       // not used beside numbers
  expect(sr_adamw_norm(t.data(), same, 6, &o, nullptr, nullptr), SR_OK, 2, "numbers alone");
  expect(sr_adamw_norm(t.data(), nullptr, 6, &o, nullptr, nullptr), SR_EINVAL, 0, "no number");
  expect(sr_adamw_norm(nullptr, nullptr, 0, &kOptions, nullptr, nullptr), SR_OK, 0, "nothing");
  expect(sr_adamw_norm(nullptr, none, 0, &kOptions, nullptr, nullptr), SR_OK, 0, "nothing, with numbers");
}

// Launches of the largest arrays: grids stay below 2^32 threads, and the tables
// name every element once.
void expect_grids(const char* what) {
  for (const model::Launch& l : launches)
    if (l.blocks == 0 || l.blocks * l.threads >= uint64_t(1) << 32) {
      std::printf("a grid of %llu blocks of %llu\n", (unsigned long long)l.blocks, (unsigned long long)l.threads);
      die(what);
    }
}

void grids() {
  const uint64_t most = SR_STEP_MAX_ELEMENTS, far = uint64_t(1) << 37;
  const std::vector<std::vector<uint64_t>> lists = {
      {most}, {most - 1}, {most - 2048 * 7}, {most - 2048 * 8}, {most / 2}, {most / 2 + 1}, {5, most, 2049},
      {most / 2 - 1, most / 2}, std::vector<uint64_t>(16, most / 16), std::vector<uint64_t>(17, most / 16)};
  for (const auto& list : lists) {
    std::vector<sr_adamw_tensor> t;
    std::vector<sr_array> a;
    for (uint64_t n : list) {
      const uint64_t b = 4 * far * t.size();
      t.push_back({at(b), at(b + far), at(b + 2 * far), nullptr, at(b + 3 * far), n, SR_DT_BF16, SR_DT_BF16, SR_DT_BF16, 0});
      a.push_back({at(b), n, SR_DT_F32, 0});
    }
    const int32_t count = int32_t(t.size());
    launches.clear();
    if (sr_adamw(t.data(), count, &kOptions, nullptr, nullptr) != SR_OK) die("adamw");
    expect_grids("adamw");
    size_t tensor = 0;
    uint64_t done = 0;        // elements of it that were named
    for (size_t l = 0; l < launches.size(); ++l) {
      const AdamTable<false>& tab = table<false>(l);
      if (launches[l].blocks < tab.at.chunks) die("fewer workgroups than chunks");
      for (uint32_t e = 0; e < tab.at.count; ++e) {
        const uint32_t to = e + 1 < tab.at.count ? tab.at.first[e + 1] : tab.at.chunks;
        const uint64_t n = uint64_t(to - tab.at.first[e] - 1) * kAdamChunk + tab.tail[e];
        const sr_adamw_tensor& x = t[tensor];
        const uint64_t shift = done * 2;
        if (tab.entry[e].weight != reinterpret_cast<uint64_t>(x.weight) + shift ||
            tab.entry[e].exp_avg != reinterpret_cast<uint64_t>(x.exp_avg) + shift ||
            tab.entry[e].exp_avg_sq != reinterpret_cast<uint64_t>(x.exp_avg_sq) + shift ||
            tab.entry[e].grad != reinterpret_cast<uint64_t>(x.grad) + shift || tab.tail[e] > kAdamChunk)
          die("another place");
        done += n;
        if (done > x.n) die("beyond a tensor");
        if (done == x.n) ++tensor, done = 0;
      }
    }
    if (tensor != t.size() || done) die("elements that no launch takes");
    launches.clear();
    const sr_norm norm = own_norm();
    if (sr_clip_norm(a.data(), nullptr, count, 1.0f, &norm, nullptr) != SR_OK) die("clip");
    expect_grids("clip");
    launches.clear();
  }
}

}  // namespace

int main(int argc, char** argv) {
  const char* scenario = argc > 1 ? argv[1] : "";
  if (!std::strcmp(scenario, "refusals")) refusals();
  else if (!std::strcmp(scenario, "steps")) steps();
  else if (!std::strcmp(scenario, "grids")) grids();
  else die("no such scenario");
  std::printf("ok\n");
  return 0;
}
