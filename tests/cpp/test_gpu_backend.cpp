// GPU tests of the C++ drop-in API: the HIP TransferBackend (one kernel per
// BoundTransfer) and the shared-arena handoff connector. Scenarios follow the
// reference's test/test_page_migration_cuda.cpp:13-108 (byte fills, pending /
// failed-safe states) and test/test_serving/test_pd_handoff.cpp:429-564
// (pattern-filled pages compared element-wise after the handoff).
#include <hip/hip_runtime.h>

#include <dlfcn.h>
#include <unistd.h>

#include <algorithm>
#include <thread>
#include <chrono>
#include <cmath>
#include <atomic>
#include <memory>
#include <string>
#include <cstring>
#include <numeric>
#include <vector>

#include "cache/page_migration.h"
#include "cache/transfer_plan.h"
#include "minitest.h"
#include "pbe_handoff.h"
#include "base/shared_kv_arena.h"
#include "serving/decode_kv_reservation.h"
#include "serving/pd_handoff.h"
#include "serving/split_pd_handoff.h"
#include "base/kv_cache_manager.h"
#include "model/paged_kv_runtime.h"

using namespace cache;

#define HIP_OK(x) REQUIRE((x) == hipSuccess)

namespace {

PageSchema schema_of(bool fp8, int32_t layers = 2) {
  PageSchema s;
  MakeKVPageSchema(1, layers, 16, 2, 64,
                   base::MakeKVCacheStorageSpec(base::DataType::kDataTypeBf16,
                                                fp8 ? base::BlockStorageMode::kFp8E4M3PerTokenHead
                                                    : base::BlockStorageMode::kPlain),
                   &s);
  return s;
}

std::vector<size_t> iota_order(size_t n) {
  std::vector<size_t> o(n);
  std::iota(o.begin(), o.end(), 0);
  return o;
}

BackendResult wait_done(TransferBackend& b, MigrationId id) {
  BackendResult r = BackendResult::kPending;
  for (int i = 0; i < 2000000 && r == BackendResult::kPending; ++i) r = b.poll(id);
  return r;
}

}  // namespace

TEST_CASE("hip backend: device to device, to host and back to device") {
  for (bool fp8 : {false, true}) {
    const auto s = schema_of(fp8);
    LayoutDescriptor l;
    REQUIRE(MakePackedLayout(s, "packed", 7, iota_order(s.components.size()), {}, &l));
    const size_t n = l.total_bytes;
    uint8_t *d_src = nullptr, *d_dst = nullptr, *d_back = nullptr, *h_pin = nullptr;
    HIP_OK(hipMalloc(&d_src, n));
    HIP_OK(hipMalloc(&d_dst, n));
    HIP_OK(hipMalloc(&d_back, n));
    HIP_OK(hipHostMalloc(&h_pin, n, hipHostMallocDefault));
    std::vector<uint8_t> pattern(n);
    for (size_t i = 0; i < n; ++i) pattern[i] = static_cast<uint8_t>(i * 37u + 11u);
    HIP_OK(hipMemcpy(d_src, pattern.data(), n, hipMemcpyHostToDevice));
    HIP_OK(hipMemset(d_dst, 0x21, n));
    HIP_OK(hipMemset(d_back, 0x21, n));
    std::memset(h_pin, 0x21, n);

    TransferPlanner planner;
    TransferPlan plan;
    REQUIRE(planner.plan(s, s, &plan));
    auto backend = MakeHipTransferBackend(2, 0);
    CHECK(backend->supports(base::DeviceType::kDeviceHIP));
    CHECK(!backend->supports(base::DeviceType::kDeviceCPU));

    BoundTransfer d2d, d2h, h2d;
    REQUIRE(BoundTransfer::Bind(plan, s, {d_src, n, &l}, {d_dst, n, &l}, &d2d));
    REQUIRE(BoundTransfer::Bind(plan, s, {d_src, n, &l}, {h_pin, n, &l}, &d2h));
    REQUIRE(BoundTransfer::Bind(plan, s, {h_pin, n, &l}, {d_back, n, &l}, &h2d));

    CHECK(backend->submit(1, TransferDirection::kGpuToGpu, d2d) == BackendResult::kPending);
    CHECK(backend->submit(1, TransferDirection::kGpuToGpu, d2d) == BackendResult::kUnknown);  // live id
    CHECK(backend->submit(2, TransferDirection::kToHost, d2h) == BackendResult::kPending);
    CHECK(backend->submit(3, TransferDirection::kToHost, d2h) == BackendResult::kFailedSafe);  // no slot
    CHECK(wait_done(*backend, 1) == BackendResult::kSucceeded);
    CHECK(backend->drain(2) == BackendResult::kSucceeded);
    backend->release(1);
    backend->release(2);
    CHECK(std::memcmp(h_pin, pattern.data(), n) == 0);
    std::vector<uint8_t> got(n);
    HIP_OK(hipMemcpy(got.data(), d_dst, n, hipMemcpyDeviceToHost));
    CHECK(got == pattern);

    CHECK(backend->submit(4, TransferDirection::kToGpu, h2d) == BackendResult::kPending);
    CHECK(backend->drain(4) == BackendResult::kSucceeded);
    backend->release(4);
    HIP_OK(hipMemcpy(got.data(), d_back, n, hipMemcpyDeviceToHost));
    CHECK(got == pattern);

    // Wrong-direction or pageable endpoints are refused before any write.
    std::vector<uint8_t> pageable(n, 0x21);
    BoundTransfer bad;
    REQUIRE(BoundTransfer::Bind(plan, s, {d_src, n, &l}, {pageable.data(), n, &l}, &bad));
    CHECK(backend->submit(5, TransferDirection::kToHost, bad) == BackendResult::kFailedSafe);
    CHECK(backend->submit(6, TransferDirection::kToGpu, d2d) == BackendResult::kFailedSafe);
    CHECK(backend->submit(7, TransferDirection::kToHost, d2d) == BackendResult::kFailedSafe);
    backend->release(5);  // never submitted to a stream: no-op
    CHECK(std::all_of(pageable.begin(), pageable.end(), [](uint8_t b) { return b == 0x21; }));
    (void)hipFree(d_src);
    (void)hipFree(d_dst);
    (void)hipFree(d_back);
    (void)hipHostFree(h_pin);
  }
}

TEST_CASE("hip backend: a dependency event orders the copy after the producer") {
  const auto s = schema_of(false);
  LayoutDescriptor l;
  REQUIRE(MakePackedLayout(s, "packed", 7, iota_order(s.components.size()), {}, &l));
  const size_t n = l.total_bytes;
  uint8_t *d_src = nullptr, *d_dst = nullptr;
  HIP_OK(hipMalloc(&d_src, n));
  HIP_OK(hipMalloc(&d_dst, n));
  hipStream_t producer;
  hipEvent_t produced;
  HIP_OK(hipStreamCreateWithFlags(&producer, hipStreamNonBlocking));
  HIP_OK(hipEventCreateWithFlags(&produced, hipEventDisableTiming));
  HIP_OK(hipMemsetAsync(d_src, 0x5c, n, producer));  // the "prefill" writes the source
  HIP_OK(hipEventRecord(produced, producer));
  TransferPlanner planner;
  TransferPlan plan;
  REQUIRE(planner.plan(s, s, &plan));
  BoundTransfer t;
  REQUIRE(BoundTransfer::Bind(plan, s, {d_src, n, &l}, {d_dst, n, &l}, &t));
  {
    auto backend = MakeHipTransferBackend(1, 0, produced);
    CHECK(backend->submit(1, TransferDirection::kGpuToGpu, t) == BackendResult::kPending);
    CHECK(backend->drain(1) == BackendResult::kSucceeded);
    backend->release(1);
  }
  std::vector<uint8_t> got(n);
  HIP_OK(hipMemcpy(got.data(), d_dst, n, hipMemcpyDeviceToHost));
  CHECK(std::all_of(got.begin(), got.end(), [](uint8_t b) { return b == 0x5c; }));
  (void)hipEventDestroy(produced);
  (void)hipStreamDestroy(producer);
  (void)hipFree(d_src);
  (void)hipFree(d_dst);
}

namespace {
// Holds a stream until the test lets it go (the gate of
// test_page_migration_cuda.cpp:8-12), with a bound so that a failed test can
// never leave the host function waiting.
std::atomic<bool> g_gate_open{false};
void hold_stream(void*) {
  const auto until = std::chrono::steady_clock::now() + std::chrono::seconds(20);
  while (!g_gate_open.load() && std::chrono::steady_clock::now() < until) std::this_thread::yield();
}
}  // namespace

TEST_CASE("hip backend: a gated dependency keeps the copy pending and its destination untouched") {
  for (bool fp8 : {false, true}) {
    const auto s = schema_of(fp8);
    LayoutDescriptor l;
    REQUIRE(MakePackedLayout(s, "packed", 7, iota_order(s.components.size()), {}, &l));
    const size_t n = l.total_bytes;
    uint8_t *d_src = nullptr, *h_dst = nullptr;
    HIP_OK(hipMalloc(&d_src, n));
    HIP_OK(hipHostMalloc(&h_dst, n, hipHostMallocDefault));  // before the gate: may synchronize
    HIP_OK(hipMemset(d_src, 0x21, n));
    std::memset(h_dst, 0, n);
    HIP_OK(hipDeviceSynchronize());
    TransferPlanner planner;
    TransferPlan plan;
    REQUIRE(planner.plan(s, s, &plan));
    BoundTransfer d2h;
    REQUIRE(BoundTransfer::Bind(plan, s, {d_src, n, &l}, {h_dst, n, &l}, &d2h));
    hipStream_t producer;
    hipEvent_t dependency;
    HIP_OK(hipStreamCreateWithFlags(&producer, hipStreamNonBlocking));
    HIP_OK(hipEventCreateWithFlags(&dependency, hipEventDisableTiming));
    {
      auto backend = MakeHipTransferBackend(1, 0, dependency);
      g_gate_open.store(false);
      const bool gated = hipLaunchHostFunc(producer, hold_stream, nullptr) == hipSuccess &&
                         hipEventRecord(dependency, producer) == hipSuccess;
      CHECK(gated);
      const BackendResult submitted = backend->submit(1, TransferDirection::kToHost, d2h);
      CHECK(submitted == BackendResult::kPending);
      if (gated && submitted == BackendResult::kPending) {
        const auto until = std::chrono::steady_clock::now() + std::chrono::milliseconds(50);
        bool pending = true;
        while (std::chrono::steady_clock::now() < until) pending = pending && backend->poll(1) == BackendResult::kPending;
        CHECK(pending);
        CHECK(std::all_of(h_dst, h_dst + n, [](uint8_t b) { return b == 0; }));
      }
      g_gate_open.store(true);  // always, whatever failed above
      HIP_OK(hipStreamSynchronize(producer));
      if (submitted == BackendResult::kPending) {
        CHECK(backend->drain(1) == BackendResult::kSucceeded);
        backend->release(1);
      }
      CHECK(std::all_of(h_dst, h_dst + n, [](uint8_t b) { return b == 0x21; }));
    }
    (void)hipEventDestroy(dependency);
    (void)hipStreamDestroy(producer);
    (void)hipFree(d_src);
    (void)hipHostFree(h_dst);
  }
}

TEST_CASE("hip backend: completion is in submission order; settled records are reused") {
  const auto s = schema_of(false, 8);
  LayoutDescriptor l;
  REQUIRE(MakePackedLayout(s, "packed", 7, iota_order(s.components.size()), {}, &l));
  const size_t n = l.total_bytes;
  std::vector<uint8_t*> bufs(4);
  for (auto& b : bufs) HIP_OK(hipMalloc(&b, n));
  HIP_OK(hipMemset(bufs[0], 0x11, n));
  HIP_OK(hipMemset(bufs[2], 0x22, n));
  TransferPlanner planner;
  TransferPlan plan;
  REQUIRE(planner.plan(s, s, &plan));
  BoundTransfer a, b;
  REQUIRE(BoundTransfer::Bind(plan, s, {bufs[0], n, &l}, {bufs[1], n, &l}, &a));
  REQUIRE(BoundTransfer::Bind(plan, s, {bufs[2], n, &l}, {bufs[3], n, &l}, &b));
  auto backend = MakeHipTransferBackend(2, 0);
  for (int round = 0; round < 3; ++round) {
    const MigrationId first = 10 + 2 * round, second = first + 1;
    CHECK(backend->submit(first, TransferDirection::kGpuToGpu, a) == BackendResult::kPending);
    CHECK(backend->submit(second, TransferDirection::kGpuToGpu, b) == BackendResult::kPending);
    CHECK(backend->drain(second) == BackendResult::kSucceeded);
    // the earlier launch finished before the later one on the same stream
    CHECK(backend->poll(first) == BackendResult::kSucceeded);
    CHECK(backend->poll(99) == BackendResult::kUnknown);
    backend->release(second);
    backend->release(first);
  }
  std::vector<uint8_t> got(n);
  HIP_OK(hipMemcpy(got.data(), bufs[1], n, hipMemcpyDeviceToHost));
  CHECK(std::all_of(got.begin(), got.end(), [](uint8_t v) { return v == 0x11; }));
  HIP_OK(hipMemcpy(got.data(), bufs[3], n, hipMemcpyDeviceToHost));
  CHECK(std::all_of(got.begin(), got.end(), [](uint8_t v) { return v == 0x22; }));
  for (auto p : bufs) (void)hipFree(p);
}

namespace {
serving::KVBlockManifest manifest_for(int32_t layers, const std::vector<int32_t>& src,
                                      const std::vector<int32_t>& dst) {
  serving::KVBlockManifest m;
  m.client_request_id.value = "req";
  m.handoff_id.value = 1;
  m.prompt_tokens = static_cast<int32_t>(src.size()) * 16;
  m.computed_tokens = m.prompt_tokens - 3;
  m.src_pool = {0, layers, 16, 2, 64, base::DataType::kDataTypeBf16, base::BlockStorageMode::kPlain};
  m.dst_pool = m.src_pool;
  for (int32_t l = 0; l < layers; ++l) m.layer_mappings.push_back({l, src, dst});
  return m;
}
}  // namespace

TEST_CASE("shared-arena connector: page-major pages arrive intact, errors write nothing") {
  const int32_t layers = 3;
  const uint64_t half = 16 * 2 * 64 * 2, page = 2 * layers * half;
  const uint64_t pages = 40, bytes = pages * page;
  pbe_arena* arena = nullptr;
  REQUIRE(pbe_arena_create(0, bytes, 0, 123, &arena) == PBE_OK);
  serving::SharedArenaBinding bind;
  REQUIRE(pbe_arena_get_view(arena, &bind.view) == PBE_OK);
  bind.epoch = 123;
  bind.device = 0;
  // Byte (2l+plane)*half of page p holds p*3 + 64*plane + l (the page-major
  // pattern of demo/shared_kv_reuse_probe.cpp:76-83).
  std::vector<uint8_t> host(bytes);
  for (uint64_t p = 0; p < pages; ++p)
    for (int l = 0; l < layers; ++l)
      for (int plane = 0; plane < 2; ++plane)
        std::memset(host.data() + p * page + (2 * l + plane) * half,
                    static_cast<int>((p * 3 + 64 * plane + l) & 0xff), half);
  HIP_OK(hipMemcpy(bind.view.base[0], host.data(), bytes, hipMemcpyHostToDevice));
  const int32_t st = 2 * layers;
  const std::vector<int32_t> src = {2 * st, 3 * st, 4 * st, 9 * st, 10 * st};
  const std::vector<int32_t> dst = {20 * st, 21 * st, 30 * st, 31 * st, 5 * st};
  {
    serving::SharedArenaKVTransferConnector conn(bind);
    serving::HandoffId h;
    REQUIRE(conn.submit(manifest_for(layers, src, dst), &h));
    CHECK(conn.drain(h).ok());
    CHECK_EQ(conn.copied_bytes(), src.size() * page);
    conn.release(h);
    CHECK(conn.poll(h).state == serving::KVTransferState::kFailed);  // forgotten

    // Errors: stale epoch, non-page-major layers, ids outside the arena.
    serving::HandoffId bad;
    CHECK(!conn.submit_from(124, manifest_for(layers, src, dst), &bad));
    CHECK(conn.poll(bad).state == serving::KVTransferState::kFailed);
    auto skew = manifest_for(layers, src, dst);
    skew.layer_mappings[1].src_block_ids[0] += st;
    CHECK(!conn.submit(skew, &bad));
    auto out_of_arena = manifest_for(layers, src, {20 * st, 21 * st, 30 * st, 31 * st, 40 * st});
    CHECK(!conn.submit(out_of_arena, &bad));
    auto unaligned = manifest_for(layers, src, {20 * st, 21 * st, 30 * st, 31 * st, 5 * st + 1});
    CHECK(!conn.submit(unaligned, &bad));
    auto self = manifest_for(layers, src, src);
    CHECK(!conn.submit(self, &bad));
  }
  std::vector<uint8_t> got(bytes);
  HIP_OK(hipMemcpy(got.data(), bind.view.base[0], bytes, hipMemcpyDeviceToHost));
  std::vector<uint8_t> want = host;
  for (size_t i = 0; i < src.size(); ++i)
    std::memcpy(want.data() + (uint64_t)dst[i] / st * page, host.data() + (uint64_t)src[i] / st * page, page);
  CHECK(got == want);
  CHECK(pbe_arena_destroy(arena) == PBE_OK);
}

TEST_CASE("generic plan form: InProcKVBlockCopyConnector equals the run copy, BF16 and FP8 pools") {
  for (bool fp8 : {false, true}) {
    const int layers = 4;
    const uint64_t elem = fp8 ? 1 : 2;
    const uint64_t half = 16 * 2 * 64 * elem, page = 2 * layers * half, pages = 24;
    const uint64_t bytes = pages * page;
    const uint64_t scale_page = 2 * layers * 16 * 2 * 4;
    uint8_t *arena = nullptr, *scales = nullptr;
    HIP_OK(hipMalloc(&arena, bytes));
    HIP_OK(hipMalloc(&scales, pages * scale_page));
    std::vector<uint8_t> host(bytes), host_sc(pages * scale_page);
    for (size_t i = 0; i < host.size(); ++i) host[i] = static_cast<uint8_t>(i * 131u + 17u);
    for (size_t i = 0; i < host_sc.size(); ++i) host_sc[i] = static_cast<uint8_t>(i * 7u + 3u);
    HIP_OK(hipMemcpy(arena, host.data(), bytes, hipMemcpyHostToDevice));
    HIP_OK(hipMemcpy(scales, host_sc.data(), host_sc.size(), hipMemcpyHostToDevice));
    serving::ArenaKVPool pool;
    pool.view.bytes = bytes;
    pool.view.segment_bytes = bytes;
    pool.view.nseg = 1;
    pool.view.base[0] = arena;
    pool.pool = {0, layers, 16, 2, 64, base::DataType::kDataTypeBf16,
                 fp8 ? base::BlockStorageMode::kFp8E4M3PerTokenHead : base::BlockStorageMode::kPlain};
    if (fp8) {
      pool.scales = scales;
      pool.scale_bytes = pages * scale_page;
    }
    const int st = 2 * layers;
    const std::vector<int32_t> src = {1 * st, 2 * st, 3 * st, 7 * st, 9 * st};
    const std::vector<int32_t> dst = {10 * st, 11 * st, 20 * st, 21 * st, 22 * st};
    const std::vector<int32_t> src2 = {4 * st, 5 * st, 6 * st};
    const std::vector<int32_t> dst2 = {13 * st, 14 * st, 15 * st};
    serving::KVBlockManifest m;
    m.client_request_id.value = "g";
    m.handoff_id.value = 3;
    m.prompt_tokens = m.computed_tokens = 80;
    m.src_pool = m.dst_pool = pool.pool;
    for (int l = 0; l < layers; ++l) m.layer_mappings.push_back({l, src, dst});
    {
      serving::InProcKVBlockCopyConnector conn(pool, pool, 0);
      serving::HandoffId h;
      REQUIRE(conn.submit(m, &h));
      CHECK(conn.drain(h).ok());
      CHECK_EQ(conn.last_op_count(), src.size() * 2 * layers * (fp8 ? 2 : 1));
      conn.release(h);
      // Later handoffs reuse the binding the first one made: another plan
      // with another page count, then manifests the binding must still refuse
      // (a bad id on the first page or a later one, a missing layer).
      serving::KVBlockManifest m2 = m;
      for (auto& lm : m2.layer_mappings) lm = {lm.layer_idx, src2, dst2};
      REQUIRE(conn.submit(m2, &h));
      CHECK(conn.drain(h).ok());
      CHECK_EQ(conn.last_op_count(), src2.size() * 2 * layers * (fp8 ? 2 : 1));
      conn.release(h);
      serving::HandoffId bad;
      for (const auto& ids : {std::vector<int32_t>{99 * st, 14 * st, 15 * st},
                              std::vector<int32_t>{13 * st, 14 * st, 5 * st + 1}}) {
        serving::KVBlockManifest mb = m;
        for (auto& lm : mb.layer_mappings) lm = {lm.layer_idx, src2, ids};
        CHECK(!conn.submit(mb, &bad));
        CHECK(conn.poll(bad).state == serving::KVTransferState::kFailed);
      }
      serving::KVBlockManifest short_layers = m2;
      short_layers.layer_mappings.pop_back();
      CHECK(!conn.submit(short_layers, &bad));
    }
    std::vector<uint8_t> got(bytes), got_sc(host_sc.size());
    HIP_OK(hipMemcpy(got.data(), arena, bytes, hipMemcpyDeviceToHost));
    HIP_OK(hipMemcpy(got_sc.data(), scales, got_sc.size(), hipMemcpyDeviceToHost));
    std::vector<uint8_t> want = host, want_sc = host_sc;
    for (const auto& [from, to] : {std::make_pair(src, dst), std::make_pair(src2, dst2)})
      for (size_t i = 0; i < from.size(); ++i) {
        std::memcpy(want.data() + to[i] / st * page, host.data() + from[i] / st * page, page);
        if (fp8)
          std::memcpy(want_sc.data() + to[i] / st * scale_page, host_sc.data() + from[i] / st * scale_page,
                      scale_page);
      }
    CHECK(got == want);
    CHECK(got_sc == want_sc);
    (void)hipFree(arena);
    (void)hipFree(scales);
  }
}

namespace {
// The CPU oracle (oracle/liboracle.so, test infrastructure): the whole data
// effect of copy_shared_kv on a host copy of the arena.
using OracleCopy = uint64_t (*)(uint8_t*, const int32_t*, const int32_t*, int64_t, uint64_t, int32_t,
                                int32_t*, int32_t*, int32_t*);
OracleCopy oracle_copy_handoff() {
  static OracleCopy fn = [] {
    std::string self(4096, '\0');
    const ssize_t n = readlink("/proc/self/exe", &self[0], self.size());
    self.resize(n > 0 ? n : 0);
    const std::string dir = self.substr(0, self.rfind('/'));  // .../paged-batch-engine_amd/lib
    void* h = dlopen((dir + "/../../oracle/liboracle.so").c_str(), RTLD_NOW);
    return h ? reinterpret_cast<OracleCopy>(dlsym(h, "orc_copy_handoff")) : nullptr;
  }();
  return fn;
}

std::unique_ptr<base::KVCacheManager> manager_over(const std::shared_ptr<base::SharedKVPageGroup>& g,
                                                   int32_t heads, int32_t dim) {
  std::vector<std::unique_ptr<base::BlockAllocator>> layers;
  for (int l = 0; l < g->layers(); ++l)
    layers.push_back(std::make_unique<base::BlockAllocator>(16, heads, dim, g, l));
  return std::make_unique<base::KVCacheManager>(16, g->layers(), std::move(layers));
}

uint8_t* at(const pbe_arena_view& v, uint64_t off) {
  return static_cast<uint8_t*>(v.base[off / v.segment_bytes]) + off % v.segment_bytes;
}
}  // namespace

TEST_CASE("end to end: the reference's copy_shared_kv call order over KVCacheManager, bit-exact") {
  // Qwen2.5-0.5B geometry: 24 layers, 2 KV heads x 64, 16-token pages (192 KiB),
  // a 4-segment arena. Prefill and decode each own a KVCacheManager over their
  // page group, built as the reference builds the shared-arena allocators.
  const int layers = 24;
  const uint64_t half = 16 * 2 * 64 * 2, page = 2 * layers * half;
  const uint64_t arena_bytes = 64 * page;
  REQUIRE(oracle_copy_handoff() != nullptr);
  pbe_arena* arena = nullptr;
  REQUIRE(pbe_arena_create(0, arena_bytes, 16 * page, 4242, &arena) == PBE_OK);
  pbe_arena_view view{};
  REQUIRE(pbe_arena_get_view(arena, &view) == PBE_OK);
  auto owner = std::make_shared<base::LocalChunkOwner>(arena_bytes, 4242);
  owner->register_model("prefill", 24 * page);
  owner->register_model("decode", 40 * page);
  void* p_stream = nullptr;
  void* d_stream = nullptr;
  REQUIRE(pbe_stream_create(0, &p_stream) == PBE_OK);
  REQUIRE(pbe_stream_create(0, &d_stream) == PBE_OK);
  {
    auto p_client = std::make_shared<base::SharedKVArenaClient>(owner, view, "prefill", 24 * page, 0);
    auto d_client = std::make_shared<base::SharedKVArenaClient>(owner, view, "decode", 40 * page, 0);
    auto p_pages = std::make_shared<base::SharedKVPageGroup>(p_client, layers, half, 2 * 1024 * 1024, p_stream);
    auto d_pages = std::make_shared<base::SharedKVPageGroup>(d_client, layers, half, 2 * 1024 * 1024, d_stream);
    auto p_kv = manager_over(p_pages, 2, 64);
    auto d_kv = manager_over(d_pages, 2, 64);
    // a decode request already holding 2 pages, so the handoff's pages are
    // not the arena's first ones on the decode side either
    const base::RequestId other = d_kv->register_request();
    REQUIRE(d_kv->append_slots(other, 20));
    // prefill: a 41-token prompt = 3 pages, every layer
    const base::RequestId pr = p_kv->register_request();
    REQUIRE(p_kv->append_slots(pr, 41));
    // every arena byte random (canaries included)
    std::vector<uint8_t> host(arena_bytes);
    uint64_t x = 0x9e3779b97f4a7c15ull;
    for (auto& b : host) { x ^= x << 13; x ^= x >> 7; x ^= x << 17; b = static_cast<uint8_t>(x >> 24); }
    for (uint32_t s = 0; s < view.nseg; ++s)
      HIP_OK(hipMemcpy(view.base[s], host.data() + s * view.segment_bytes, view.segment_bytes, hipMemcpyHostToDevice));
    serving::KVPoolDescriptor pool{0, layers, 16, 2, 64, base::DataType::kDataTypeBf16,
                                   base::BlockStorageMode::kPlain};
    serving::SharedKVPrefillResult result;
    result.shared_arena_epoch = p_client->epoch();
    result.client_request_id.value = "req-41";
    result.handoff_id.value = 1;
    result.prompt_tokens.assign(41, 7);
    result.computed_tokens = 41;
    result.first_token = 99;
    result.src_pool = pool;
    for (int l = 0; l < layers; ++l) result.layers.push_back({l, p_kv->get_block_ids(pr, l)});
    // rejected inputs reserve nothing and write nothing
    serving::DecodeKVReservation res;
    auto bad = result;
    bad.shared_arena_epoch = 7;
    CHECK_THROWS_AS(serving::CopySharedKVToDecode(d_kv.get(), pool, bad, d_stream, &res), std::runtime_error);
    bad = result;
    bad.layers.pop_back();
    CHECK_THROWS_AS(serving::CopySharedKVToDecode(d_kv.get(), pool, bad, d_stream, &res), std::runtime_error);
    bad = result;
    bad.layers[5].src_block_ids[1] += 1;  // not a page id
    CHECK_THROWS_AS(serving::CopySharedKVToDecode(d_kv.get(), pool, bad, d_stream, &res), std::runtime_error);
    bad = result;
    bad.computed_tokens = 60;  // more than the prompt
    CHECK_THROWS_AS(serving::CopySharedKVToDecode(d_kv.get(), pool, bad, d_stream, &res), std::runtime_error);
    CHECK_EQ(d_kv->num_active_requests(), 1);
    CHECK(!res.valid());
    // reserve -> manifest -> one-launch copy -> sync -> commit_kv
    const uint64_t copied = serving::CopySharedKVToDecode(d_kv.get(), pool, result, d_stream, &res);
    CHECK_EQ(copied, 3 * page);
    REQUIRE(res.valid());
    CHECK_EQ(d_kv->kv_committed_tokens(res.decode_request_id), 41);
    CHECK_EQ(d_kv->get_context_len(res.decode_request_id), 41);
    const auto& src = p_kv->get_block_ids(pr, 0);
    const auto& dst = d_kv->get_block_ids(res.decode_request_id, 0);
    REQUIRE(dst.size() == 3u);
    CHECK(dst == res.dst_block_ids_per_layer[0]);
    CHECK(dst[0] != src[0]);
    std::vector<int32_t> s1(3), s2(3), s3(3);
    CHECK_EQ(oracle_copy_handoff()(host.data(), src.data(), dst.data(), 3, half, layers, s1.data(),
                                   s2.data(), s3.data()),
             3 * page);
    std::vector<uint8_t> got(arena_bytes);
    for (uint32_t s = 0; s < view.nseg; ++s)
      HIP_OK(hipMemcpy(got.data() + s * view.segment_bytes, view.base[s], view.segment_bytes, hipMemcpyDeviceToHost));
    CHECK(std::memcmp(got.data(), host.data(), arena_bytes) == 0);
    // copy_block_payload in shared-arena mode: one block of one layer, on the
    // group's stream (K and V planes of layer 3 of dst[0] onto dst[1])
    d_kv->allocator(3).copy_block_payload(dst[0], dst[1]);
    for (int plane = 0; plane < 2; ++plane)
      std::memcpy(host.data() + (dst[1] + 6 + plane) * half, host.data() + (dst[0] + 6 + plane) * half, half);
    for (uint32_t s = 0; s < view.nseg; ++s)
      HIP_OK(hipMemcpy(got.data() + s * view.segment_bytes, view.base[s], view.segment_bytes, hipMemcpyDeviceToHost));
    CHECK(std::memcmp(got.data(), host.data(), arena_bytes) == 0);
    (void)at;
    // prefill frees its request; the pages return once its stream passes the fences
    p_kv->free_request(pr);
    REQUIRE(pbe_stream_synchronize(0, p_stream) == PBE_OK);
    p_pages->collect();
    CHECK_EQ(p_pages->leased_bytes(), 0u);
    d_kv->free_request(res.decode_request_id);
    d_kv->free_request(other);
    REQUIRE(pbe_stream_synchronize(0, d_stream) == PBE_OK);
    d_pages->collect();
    CHECK_EQ(d_pages->leased_bytes(), 0u);
  }
  CHECK_EQ(owner->lease_count(), 0u);
  CHECK_EQ(owner->free_bytes(), arena_bytes);
  pbe_stream_destroy(0, p_stream);
  pbe_stream_destroy(0, d_stream);
  CHECK(pbe_arena_destroy(arena) == PBE_OK);
}

TEST_CASE("end to end at config-2 size: 315 pages x 28 layers through CopySharedKVToDecode, bit-exact") {
  // Qwen2.5-1.5B geometry: 28 layers, 2 KV heads x 128, 16-token pages
  // (448 KiB). A 5040-token prefill (315 pages) handed to a decode group
  // whose free pages are fragmented by earlier requests, twice in a row (the
  // second handoff reuses the first one's pages after their fences pass).
  const int layers = 28;
  const uint64_t half = 16 * 2 * 128 * 2, page = 2 * layers * half;
  const uint64_t n_pages = 760, arena_bytes = n_pages * page;
  REQUIRE(oracle_copy_handoff() != nullptr);
  pbe_arena* arena = nullptr;
  REQUIRE(pbe_arena_create(0, arena_bytes, 0, 5151, &arena) == PBE_OK);
  pbe_arena_view view{};
  REQUIRE(pbe_arena_get_view(arena, &view) == PBE_OK);
  REQUIRE(view.nseg == 1u);
  auto owner = std::make_shared<base::LocalChunkOwner>(arena_bytes, 5151);
  owner->register_model("prefill", 330 * page);
  owner->register_model("decode", 430 * page);
  void* p_stream = nullptr;
  void* d_stream = nullptr;
  REQUIRE(pbe_stream_create(0, &p_stream) == PBE_OK);
  REQUIRE(pbe_stream_create(0, &d_stream) == PBE_OK);
  {
    auto p_client = std::make_shared<base::SharedKVArenaClient>(owner, view, "prefill", 330 * page, 0);
    auto d_client = std::make_shared<base::SharedKVArenaClient>(owner, view, "decode", 430 * page, 0);
    auto p_pages = std::make_shared<base::SharedKVPageGroup>(p_client, layers, half, 2 * 1024 * 1024, p_stream);
    auto d_pages = std::make_shared<base::SharedKVPageGroup>(d_client, layers, half, 2 * 1024 * 1024, d_stream);
    auto p_kv = manager_over(p_pages, 2, 128);
    auto d_kv = manager_over(d_pages, 2, 128);
    // decode side: five requests, then every other one freed -> holes
    std::vector<base::RequestId> held;
    for (int k = 0; k < 5; ++k) {
      held.push_back(d_kv->register_request());
      REQUIRE(d_kv->append_slots(held.back(), 16 * (7 + 5 * k)));
    }
    d_kv->free_request(held[0]);
    d_kv->free_request(held[2]);
    d_kv->free_request(held[4]);
    REQUIRE(pbe_stream_synchronize(0, d_stream) == PBE_OK);
    const base::RequestId pr = p_kv->register_request();
    REQUIRE(p_kv->append_slots(pr, 5040));
    serving::KVPoolDescriptor pool{0, layers, 16, 2, 128, base::DataType::kDataTypeBf16,
                                   base::BlockStorageMode::kPlain};
    serving::SharedKVPrefillResult result;
    result.shared_arena_epoch = p_client->epoch();
    result.client_request_id.value = "req-5040";
    result.handoff_id.value = 2;
    result.prompt_tokens.assign(5040, 7);
    result.computed_tokens = 5040;
    result.first_token = 11;
    result.src_pool = pool;
    for (int l = 0; l < layers; ++l) result.layers.push_back({l, p_kv->get_block_ids(pr, l)});
    std::vector<uint8_t> host(arena_bytes), got(arena_bytes);
    uint64_t x = 0x2545f4914f6cdd1dull;
    for (uint64_t i = 0; i < arena_bytes / 8; ++i) {
      x ^= x << 13; x ^= x >> 7; x ^= x << 17;
      std::memcpy(host.data() + 8 * i, &x, 8);
    }
    HIP_OK(hipMemcpy(view.base[0], host.data(), arena_bytes, hipMemcpyHostToDevice));
    const auto& src = p_kv->get_block_ids(pr, 0);
    REQUIRE(src.size() == 315u);
    for (int round = 0; round < 2; ++round) {
      std::printf("  handoff %d\n", round);
      std::fflush(stdout);
      serving::DecodeKVReservation res;
      const uint64_t copied = serving::CopySharedKVToDecode(d_kv.get(), pool, result, d_stream, &res);
      CHECK_EQ(copied, 315 * page);
      REQUIRE(res.valid());
      CHECK_EQ(d_kv->kv_committed_tokens(res.decode_request_id), 5040);
      const auto& dst = d_kv->get_block_ids(res.decode_request_id, 0);
      REQUIRE(dst.size() == 315u);
      for (int l = 1; l < layers; ++l) CHECK(d_kv->get_block_ids(res.decode_request_id, l) == dst);
      // the destination is fragmented: it starts in the holes left above
      int runs = 1;
      for (size_t i = 1; i < dst.size(); ++i) runs += dst[i] != dst[i - 1] + 2 * layers;
      CHECK(runs > 1);
      std::vector<int32_t> s1(315), s2(315), s3(315);
      CHECK_EQ(oracle_copy_handoff()(host.data(), src.data(), dst.data(), 315, half, layers, s1.data(),
                                     s2.data(), s3.data()),
               315 * page);
      HIP_OK(hipMemcpy(got.data(), view.base[0], arena_bytes, hipMemcpyDeviceToHost));
      CHECK(std::memcmp(got.data(), host.data(), arena_bytes) == 0);
      d_kv->free_request(res.decode_request_id);
      REQUIRE(pbe_stream_synchronize(0, d_stream) == PBE_OK);
    }
    p_kv->free_request(pr);
    d_kv->free_request(held[1]);
    d_kv->free_request(held[3]);
    REQUIRE(pbe_stream_synchronize(0, p_stream) == PBE_OK);
    REQUIRE(pbe_stream_synchronize(0, d_stream) == PBE_OK);
    p_pages->collect();
    d_pages->collect();
    CHECK_EQ(p_pages->leased_bytes(), 0u);
    CHECK_EQ(d_pages->leased_bytes(), 0u);
  }
  CHECK_EQ(owner->lease_count(), 0u);
  pbe_stream_destroy(0, p_stream);
  pbe_stream_destroy(0, d_stream);
  CHECK(pbe_arena_destroy(arena) == PBE_OK);
}

TEST_CASE("page group: a retired page is not handed out again until its fence has passed") {
  // The deferred unpin of shared_kv_reuse_probe.cpp, with the stream held by
  // a host-function gate: the page's fence is queued behind the gate.
  const int layers = 2;
  const uint64_t half = 16 * 2 * 64 * 2, page = 2 * layers * half, arena_bytes = 12 * page;
  pbe_arena* arena = nullptr;
  REQUIRE(pbe_arena_create(0, arena_bytes, arena_bytes, 515, &arena) == PBE_OK);
  pbe_arena_view view{};
  REQUIRE(pbe_arena_get_view(arena, &view) == PBE_OK);
  auto owner = std::make_shared<base::LocalChunkOwner>(arena_bytes, 515);
  owner->register_model("m", arena_bytes);
  hipStream_t stream;
  HIP_OK(hipStreamCreateWithFlags(&stream, hipStreamNonBlocking));
  {
    auto client = std::make_shared<base::SharedKVArenaClient>(owner, view, "m", arena_bytes, 0);
    auto group = std::make_shared<base::SharedKVPageGroup>(client, layers, half, 3 * page, stream);
    const int a = group->allocate(0);
    REQUIRE(a >= 0);
    CHECK_EQ(group->allocate(1), a);
    g_gate_open.store(false);
    const bool gated = hipLaunchHostFunc(stream, hold_stream, nullptr) == hipSuccess;
    CHECK(gated);
    group->retire(1, a);
    group->retire(0, a);  // the last layer: the fence is recorded behind the gate
    group->collect();
    const int b = group->allocate(0);
    CHECK(b >= 0);
    CHECK(b != a);  // a is still fenced
    group->allocate(1);
    g_gate_open.store(true);  // always, whatever failed above
    HIP_OK(hipStreamSynchronize(stream));
    group->collect();
    const int c = group->allocate(0);  // the lowest free id again
    CHECK_EQ(c, a);
    group->allocate(1);
    for (int id : {b, c}) {
      group->retire(1, id);
      group->retire(0, id);
    }
    HIP_OK(hipStreamSynchronize(stream));
    group->collect();
    CHECK_EQ(group->leased_bytes(), 0u);
  }
  (void)hipStreamDestroy(stream);
  CHECK(pbe_arena_destroy(arena) == PBE_OK);
}

TEST_CASE("page group: a request's pages freed together share one fence; none is reused before it") {
  const int layers = 3;
  const uint64_t half = 16 * 2 * 64 * 2, page = 2 * layers * half, arena_bytes = 24 * page;
  pbe_arena* arena = nullptr;
  REQUIRE(pbe_arena_create(0, arena_bytes, arena_bytes, 516, &arena) == PBE_OK);
  pbe_arena_view view{};
  REQUIRE(pbe_arena_get_view(arena, &view) == PBE_OK);
  auto owner = std::make_shared<base::LocalChunkOwner>(arena_bytes, 516);
  owner->register_model("m", arena_bytes);
  void* stream = nullptr;
  REQUIRE(pbe_stream_create(0, &stream) == PBE_OK);
  {
    auto client = std::make_shared<base::SharedKVArenaClient>(owner, view, "m", arena_bytes, 0);
    auto group = std::make_shared<base::SharedKVPageGroup>(client, layers, half, 3 * page, stream);
    auto kv = manager_over(group, 2, 64);
    const base::RequestId first = kv->register_request();
    REQUIRE(kv->append_slots(first, 5 * 16));
    const std::vector<int32_t> held = kv->get_block_ids(first, 0);
    REQUIRE(held.size() == 5u);
    g_gate_open.store(false);
    CHECK(hipLaunchHostFunc(static_cast<hipStream_t>(stream), hold_stream, nullptr) == hipSuccess);
    kv->free_request(first);  // every layer; the fence lands behind the gate
    const base::RequestId second = kv->register_request();
    REQUIRE(kv->append_slots(second, 5 * 16));
    const std::vector<int32_t> fresh = kv->get_block_ids(second, 0);
    for (int32_t id : fresh) CHECK(std::find(held.begin(), held.end(), id) == held.end());
    for (int l = 1; l < layers; ++l) CHECK(kv->get_block_ids(second, l) == fresh);
    g_gate_open.store(true);  // always, whatever failed above
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    group->collect();
    // every page the second request does not hold, the first request's among them
    const base::RequestId third = kv->register_request();
    REQUIRE(kv->append_slots(third, 19 * 16));
    const std::vector<int32_t>& rest = kv->get_block_ids(third, 0);
    for (int32_t id : held) CHECK(std::find(rest.begin(), rest.end(), id) != rest.end());
    kv->free_request(second);
    kv->free_request(third);
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    group->collect();
    CHECK_EQ(group->leased_bytes(), 0u);
  }
  pbe_stream_destroy(0, stream);
  CHECK(pbe_arena_destroy(arena) == PBE_OK);
}

TEST_CASE("block allocator: local HIP pools copy one block's payload, FP8 scales included") {
  for (int fp8 = 0; fp8 < 2; ++fp8) {
    base::BlockAllocator a(8, 16, 2, 64, base::DataType::kDataTypeBf16, base::DeviceType::kDeviceHIP,
                           fp8 ? base::BlockStorageMode::kFp8E4M3PerTokenHead : base::BlockStorageMode::kPlain);
    CHECK_EQ(a.key_value_bytes_per_block(), fp8 ? 2048u : 4096u);
    CHECK_EQ(a.scale_bytes_per_block(), fp8 ? 128u : 0u);
    int ids[8];
    for (int i = 0; i < 8; ++i) ids[i] = a.allocate();
    const base::KVPoolView v = a.pool_view();
    const size_t kvb = 8 * a.key_value_bytes_per_block(), scb = 8 * a.scale_bytes_per_block();
    // random pools (payload and scales)
    std::vector<std::vector<uint8_t>> host;
    void* pools[4] = {v.key_pool(), v.value_pool(), v.key_scale_pool(), v.value_scale_pool()};
    const size_t sizes[4] = {kvb, kvb, scb, scb};
    uint64_t x = 12345 + fp8;
    for (int p = 0; p < 4; ++p) {
      host.emplace_back(sizes[p]);
      for (auto& b : host.back()) { x ^= x << 13; x ^= x >> 7; x ^= x << 17; b = static_cast<uint8_t>(x >> 32); }
      if (sizes[p]) HIP_OK(hipMemcpy(pools[p], host[p].data(), sizes[p], hipMemcpyHostToDevice));
    }
    a.copy_block_payload(ids[5], ids[2]);
    const size_t per[4] = {a.key_value_bytes_per_block(), a.key_value_bytes_per_block(),
                           a.scale_bytes_per_block(), a.scale_bytes_per_block()};
    for (int p = 0; p < 4; ++p) {
      if (!sizes[p]) continue;
      std::memcpy(host[p].data() + ids[2] * per[p], host[p].data() + ids[5] * per[p], per[p]);
      std::vector<uint8_t> got(sizes[p]);
      HIP_OK(hipMemcpy(got.data(), pools[p], sizes[p], hipMemcpyDeviceToHost));
      CHECK(got == host[p]);
    }
    CHECK_EQ(a.payload_copy_bytes(), 2 * per[0] + 2 * per[2]);
    CHECK_THROWS_AS(a.copy_block_payload(ids[1], ids[1]), std::logic_error);
  }
}

TEST_CASE("interprocess events: unsupported runtimes say so at create, in-process events work") {
  pbe_event* ev = nullptr;
  const int rc = pbe_event_create(0, 1, &ev);
  if (rc == PBE_ERR_UNSUPPORTED) {
    CHECK(ev == nullptr);
    CHECK(std::string(pbe_last_error()).find("pbe_signal_") != std::string::npos);
    uint8_t handle[PBE_IPC_HANDLE_BYTES] = {};
    pbe_event* imported = nullptr;
    CHECK_EQ(pbe_event_import(handle, 0, &imported), PBE_ERR_UNSUPPORTED);
  } else {
    // a runtime that records interprocess events: export, import, record, wait
    REQUIRE(rc == PBE_OK);
    uint8_t handle[PBE_IPC_HANDLE_BYTES];
    REQUIRE(pbe_event_export(ev, handle) == PBE_OK);
    pbe_event* imported = nullptr;
    REQUIRE(pbe_event_import(handle, 0, &imported) == PBE_OK);
    REQUIRE(pbe_event_record(ev, nullptr) == PBE_OK);
    REQUIRE(pbe_event_wait(imported, nullptr) == PBE_OK);
    REQUIRE(pbe_event_synchronize(ev) == PBE_OK);
    pbe_event_destroy(imported);
    pbe_event_destroy(ev);
  }
  pbe_event* local = nullptr;
  REQUIRE(pbe_event_create(0, 0, &local) == PBE_OK);
  uint8_t handle[PBE_IPC_HANDLE_BYTES];
  CHECK_EQ(pbe_event_export(local, handle), PBE_ERR_INVALID);
  REQUIRE(pbe_event_record(local, nullptr) == PBE_OK);
  CHECK_EQ(pbe_event_synchronize(local), PBE_OK);
  CHECK_EQ(pbe_event_query(local), PBE_OK);
  pbe_event_destroy(local);
}

TEST_CASE("zero-copy takeover: moved Chunks are read in place, shared pages are copied") {
  // Qwen2.5-0.5B geometry, 3-page Chunks: request A = 5 pages, request B = 1
  // page in A's last Chunk, so A's pages 3-4 must be copied and 0-2 move.
  const int layers = 24;
  const uint64_t half = 16 * 2 * 64 * 2, page = 2 * layers * half;
  const uint64_t arena_bytes = 48 * page;
  pbe_arena* arena = nullptr;
  REQUIRE(pbe_arena_create(0, arena_bytes, 16 * page, 5151, &arena) == PBE_OK);  // 3 segments
  pbe_arena_view view{};
  REQUIRE(pbe_arena_get_view(arena, &view) == PBE_OK);
  auto owner = std::make_shared<base::LocalChunkOwner>(arena_bytes, 5151);
  owner->register_model("prefill", 24 * page);
  owner->register_model("decode", 24 * page);
  void* p_stream = nullptr;
  void* d_stream = nullptr;
  REQUIRE(pbe_stream_create(0, &p_stream) == PBE_OK);
  REQUIRE(pbe_stream_create(0, &d_stream) == PBE_OK);
  auto addr = [&](int32_t id) {
    const uint64_t off = static_cast<uint64_t>(id) * half;
    return static_cast<uint8_t*>(view.base[off / view.segment_bytes]) + off % view.segment_bytes;
  };
  {
    auto p_client = std::make_shared<base::SharedKVArenaClient>(owner, view, "prefill", 24 * page, 0);
    auto d_client = std::make_shared<base::SharedKVArenaClient>(owner, view, "decode", 24 * page, 0);
    base::SharedKVPageGroup p_pages(p_client, layers, half, 3 * page, p_stream);
    base::SharedKVPageGroup d_pages(d_client, layers, half, 3 * page, d_stream);
    auto alloc = [&](int n) {
      std::vector<int32_t> ids;
      for (int i = 0; i < n; ++i) ids.push_back(p_pages.allocate(0));
      for (int l = 1; l < layers; ++l)
        for (int i = 0; i < n; ++i) CHECK_EQ(p_pages.allocate(l), ids[i]);
      return ids;
    };
    auto a = alloc(5);
    auto b = alloc(1);
    std::vector<uint8_t> host(page);
    for (size_t i = 0; i < a.size(); ++i) {
      for (uint64_t k = 0; k < page; ++k) host[k] = static_cast<uint8_t>((k * 7 + i * 31) >> 3);
      HIP_OK(hipMemcpy(addr(a[i]), host.data(), page, hipMemcpyHostToDevice));
    }
    base::SharedKVPageGroup::PageTakeover tk;
    p_pages.detach_for_takeover(a, &tk);
    CHECK_EQ(tk.moved_ids.size(), 3u);
    CHECK_EQ(tk.copy_ids.size(), 2u);
    serving::KVPoolDescriptor pool{0, layers, 16, 2, 64, base::DataType::kDataTypeBf16,
                                   base::BlockStorageMode::kPlain};
    serving::SharedArenaBinding binding{view, 5151, 0};
    std::vector<int32_t> table;
    uint64_t copied = 0;
    REQUIRE(serving::TakeOverSharedKV(&d_pages, binding, tk, pool, d_stream, &table, &copied));
    p_pages.finish_takeover(tk);
    CHECK_EQ(copied, 2 * page);
    REQUIRE(table.size() == a.size());
    for (int i = 0; i < 3; ++i) CHECK_EQ(table[i], a[i]);  // used in place
    REQUIRE(pbe_stream_synchronize(0, d_stream) == PBE_OK);
    for (size_t i = 0; i < a.size(); ++i) {
      HIP_OK(hipMemcpy(host.data(), addr(table[i]), page, hipMemcpyDeviceToHost));
      bool ok = true;
      for (uint64_t k = 0; k < page && ok; ++k) ok = host[k] == static_cast<uint8_t>((k * 7 + i * 31) >> 3);
      CHECK(ok);
    }
    CHECK_EQ(owner->leased_bytes("decode"), 6 * page);  // adopted Chunk + a Chunk for the 2 copies
    CHECK_EQ(owner->leased_bytes("prefill"), 3 * page);
    // prefill retires the copied pages and B; decode retires the whole request
    for (int l = 0; l < layers; ++l) {
      for (int32_t id : tk.copy_ids) p_pages.retire(l, id);
      for (int32_t id : b) p_pages.retire(l, id);
      for (int32_t id : table) d_pages.retire(l, id);
    }
    REQUIRE(pbe_stream_synchronize(0, p_stream) == PBE_OK);
    REQUIRE(pbe_stream_synchronize(0, d_stream) == PBE_OK);
    p_pages.collect();
    d_pages.collect();
    CHECK_EQ(p_pages.leased_bytes(), 0u);
    CHECK_EQ(d_pages.leased_bytes(), 0u);
  }
  CHECK_EQ(owner->lease_count(), 0u);
  CHECK_EQ(owner->free_bytes(), arena_bytes);
  pbe_stream_destroy(0, p_stream);
  pbe_stream_destroy(0, d_stream);
  CHECK(pbe_arena_destroy(arena) == PBE_OK);
}

namespace {
// orc_scatter_kv of the CPU oracle (test infrastructure), the page writer's restatement.
using OracleScatter = void (*)(const uint8_t*, const uint8_t*, int32_t, int64_t, const int32_t*, int32_t,
                               int32_t, int32_t, int32_t, uint8_t*, uint64_t, uint8_t*, uint64_t, float*,
                               uint64_t, float*, uint64_t);
OracleScatter oracle_scatter() {
  static OracleScatter fn = [] {
    std::string self(4096, '\0');
    const ssize_t n = readlink("/proc/self/exe", &self[0], self.size());
    self.resize(n > 0 ? n : 0);
    const std::string dir = self.substr(0, self.rfind('/'));
    void* h = dlopen((dir + "/../../oracle/liboracle.so").c_str(), RTLD_NOW);
    return h ? reinterpret_cast<OracleScatter>(dlsym(h, "orc_scatter_kv")) : nullptr;
  }();
  return fn;
}

std::vector<uint8_t> random_bytes(size_t n, uint64_t seed) {
  std::vector<uint8_t> v(n);
  for (auto& b : v) { seed ^= seed << 13; seed ^= seed >> 7; seed ^= seed << 17; b = static_cast<uint8_t>(seed >> 24); }
  return v;
}

// BF16 values N(0,1)-like from random bytes: keep sign and a small exponent range.
std::vector<uint8_t> random_bf16(size_t elems, uint64_t seed) {
  std::vector<uint8_t> raw = random_bytes(2 * elems, seed);
  for (size_t i = 0; i < elems; ++i) {
    uint16_t h = static_cast<uint16_t>(raw[2 * i] | (raw[2 * i + 1] << 8));
    h = static_cast<uint16_t>((h & 0x807f) | ((0x7a + (h >> 7) % 8) << 7));  // |x| in [2^-5, 2^3)
    raw[2 * i] = static_cast<uint8_t>(h);
    raw[2 * i + 1] = static_cast<uint8_t>(h >> 8);
  }
  return raw;
}

template <typename T>
T* to_device(const std::vector<T>& v) {
  T* d = nullptr;
  if (hipMalloc(&d, v.size() * sizeof(T)) != hipSuccess) return nullptr;
  if (hipMemcpy(d, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) return nullptr;
  return d;
}

std::vector<uint8_t> to_host(const void* d, size_t n) {
  std::vector<uint8_t> v(n);
  if (n && hipMemcpy(v.data(), d, n, hipMemcpyDeviceToHost) != hipSuccess) v.clear();
  return v;
}
}  // namespace

TEST_CASE("model runtime: prompt K/V written through KVCacheManager slots, then decoded from the pool views") {
  REQUIRE(oracle_scatter() != nullptr);
  const int layers = 24, H = 2, D = 64, B = 16;
  const uint64_t half = B * H * D * 2, page = 2 * layers * half, arena_bytes = 32 * page;
  void* stream = nullptr;
  REQUIRE(pbe_stream_create(0, &stream) == PBE_OK);
  const model::HipPagedKVRuntime runtime(0, stream);
  {
    // (1) shared page-major arena, BF16: the slots of a 41-token prompt of
    // layer 7, from the manager's page tables, as the model's forward builds them.
    pbe_arena* arena = nullptr;
    REQUIRE(pbe_arena_create(0, arena_bytes, arena_bytes, 77, &arena) == PBE_OK);
    pbe_arena_view view{};
    REQUIRE(pbe_arena_get_view(arena, &view) == PBE_OK);
    auto owner = std::make_shared<base::LocalChunkOwner>(arena_bytes, 77);
    owner->register_model("decode", arena_bytes);
    {
      auto client = std::make_shared<base::SharedKVArenaClient>(owner, view, "decode", arena_bytes, 0);
      auto pages = std::make_shared<base::SharedKVPageGroup>(client, layers, half, 2 * 1024 * 1024, stream);
      auto kv = manager_over(pages, H, D);
      const base::RequestId first = kv->register_request();
      REQUIRE(kv->append_slots(first, 33));  // pages ahead of the prompt's
      const base::RequestId req = kv->register_request();
      REQUIRE(kv->append_slots(req, 41));
      const int layer = 7;
      std::vector<int32_t> slots;
      for (int t = 0; t < 41; ++t) {
        const auto s = kv->get_slot(req, layer, t);
        slots.push_back(s.first * B + s.second);
      }
      std::vector<uint8_t> host = random_bytes(arena_bytes, 5);
      HIP_OK(hipMemcpy(view.base[0], host.data(), arena_bytes, hipMemcpyHostToDevice));
      const auto K = random_bf16(41 * H * D, 11), V = random_bf16(41 * H * D, 12);
      uint8_t* dK = to_device(K);
      uint8_t* dV = to_device(V);
      int32_t* dS = to_device(slots);
      REQUIRE(dK && dV && dS);
      const base::KVPoolView pool = kv->allocator(layer).pool_view();
      CHECK_EQ(pool.key_pool_bytes(), arena_bytes - 2 * layer * half);
      runtime.scatter(dK, dV, base::DataType::kDataTypeBf16, pool, dS, B, H, D, 41);
      REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
      const uint64_t k_off = 2 * layer * half, v_off = k_off + half;
      float none = 0.f;
      oracle_scatter()(K.data(), V.data(), 0, 41, slots.data(), B, H, D, 0, host.data() + k_off,
                       arena_bytes - k_off, host.data() + v_off, arena_bytes - v_off, &none, 0, &none, 0);
      CHECK(to_host(view.base[0], arena_bytes) == host);
      {
        // decode over the layer's pool view == decode over the page-major arena
        const int kvm = 6, batch = 2;
        const std::vector<base::RequestId> ids{first, req};
        const auto tables = kv->build_block_tables(ids, layer);
        const auto lens = kv->build_seq_lens(ids);
        const auto q = random_bf16(batch * kvm * H * D, 13);
        uint8_t* dq = to_device(q);
        int32_t* dt = to_device(tables.first);
        int32_t* dl = to_device(lens);
        uint8_t *out_pool = nullptr, *out_arena = nullptr, *ws = nullptr;
        const int32_t splits = 4;
        const uint64_t ws_bytes = pbe_paged_decode_workspace_bytes(batch, kvm * H, D, splits);
        HIP_OK(hipMalloc(&out_pool, q.size()));
        HIP_OK(hipMalloc(&out_arena, q.size()));
        HIP_OK(hipMalloc(&ws, ws_bytes));
        model::PagedKVDecodeRuntimeArgs a;
        a.batch_size = batch;
        a.head_num = kvm * H;
        a.head_size = D;
        a.kv_mul = kvm;
        a.max_blocks_per_seq = tables.second;
        a.block_size = B;
        a.num_kv_heads = H;
        a.queries = dq;
        a.outputs = out_pool;
        a.block_tables = dt;
        a.seq_lens = dl;
        a.workspace = ws;
        a.workspace_bytes = ws_bytes;
        a.splits = splits;
        CHECK(runtime.decode(pool, a));
        const pbe_kv_shape shape{layers, H, D, B};
        REQUIRE(pbe_paged_decode(&view, PBE_KV_BF16, nullptr, 0, &shape, layer, dq, out_arena, batch, kvm * H, dt,
                                 dl, tables.second, splits, ws, ws_bytes, 0, stream) == PBE_OK);
        REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
        const auto got = to_host(out_pool, q.size());
        CHECK(got == to_host(out_arena, q.size()));
        CHECK(std::any_of(got.begin(), got.end(), [](uint8_t b) { return b != 0; }));
        a.block_size = 32;
        CHECK(!runtime.decode(pool, a));  // not a shape the reader covers: the caller keeps its path
        a.block_size = B;
        a.kv_mul = 5;
        CHECK_THROWS_AS(runtime.decode(pool, a), std::invalid_argument);
        for (void* d : {static_cast<void*>(dq), static_cast<void*>(dt), static_cast<void*>(dl),
                        static_cast<void*>(out_pool), static_cast<void*>(out_arena), static_cast<void*>(ws)})
          HIP_OK(hipFree(d));
      }
      // a slot-less view is refused before any launch
      CHECK_THROWS_AS(runtime.scatter(dK, dV, base::DataType::kDataTypeBf16, base::KVPoolView(), dS, B, H, D,
                                      41),
                      std::invalid_argument);
      CHECK_THROWS_AS(runtime.scatter(dK, dV, base::DataType::kDataTypeInt8, pool, dS, B, H, D, 41),
                      std::invalid_argument);
      HIP_OK(hipFree(dK));
      HIP_OK(hipFree(dV));
      HIP_OK(hipFree(dS));
      kv->free_request(req);
      kv->free_request(first);
    }
    REQUIRE(pbe_arena_destroy(arena) == PBE_OK);
  }
  {
    // (2) local HIP pools with FP8 storage: a batch of tokens in shuffled
    // slots, then one more token at a host-known block and offset.
    base::BlockAllocator pools(8, B, H, D, base::DataType::kDataTypeBf16, base::DeviceType::kDeviceHIP,
                               base::BlockStorageMode::kFp8E4M3PerTokenHead);
    const base::KVPoolView pool = pools.pool_view();
    REQUIRE(pool.uses_fp8_storage());
    const size_t kvb = pool.key_pool_bytes(), scb = pool.scale_pool_bytes();
    CHECK_EQ(kvb, 8u * B * H * D);
    CHECK_EQ(scb, 8u * B * H * 4);
    std::vector<std::vector<uint8_t>> host;
    void* ptr[4] = {pool.key_pool(), pool.value_pool(), pool.key_scale_pool(), pool.value_scale_pool()};
    const size_t size[4] = {kvb, kvb, scb, scb};
    for (int p = 0; p < 4; ++p) {
      host.push_back(random_bytes(size[p], 40 + p));
      HIP_OK(hipMemcpy(ptr[p], host[p].data(), size[p], hipMemcpyHostToDevice));
    }
    const int n = 50;
    std::vector<int32_t> slots(8 * B);
    std::iota(slots.begin(), slots.end(), 0);
    uint64_t x = 99;
    for (size_t i = slots.size() - 1; i > 0; --i) {
      x ^= x << 13; x ^= x >> 7; x ^= x << 17;
      std::swap(slots[i], slots[x % (i + 1)]);
    }
    slots.resize(n);
    slots[3] = -1;
    const auto K = random_bf16(n * H * D, 21), V = random_bf16(n * H * D, 22);
    uint8_t* dK = to_device(K);
    uint8_t* dV = to_device(V);
    int32_t* dS = to_device(slots);
    REQUIRE(dK && dV && dS);
    runtime.scatter(dK, dV, base::DataType::kDataTypeBf16, pool, dS, B, H, D, n);
    runtime.scatter_single_token(dK + 7 * H * D * 2, dV + 7 * H * D * 2, base::DataType::kDataTypeBf16, pool, 2, 9,
                                 B, H, D);
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    auto* ks = reinterpret_cast<float*>(host[2].data());
    auto* vs = reinterpret_cast<float*>(host[3].data());
    oracle_scatter()(K.data(), V.data(), 0, n, slots.data(), B, H, D, 1, host[0].data(), kvb, host[1].data(), kvb,
                     ks, scb / 4, vs, scb / 4);
    const int32_t one = 2 * B + 9;
    oracle_scatter()(K.data() + 7 * H * D * 2, V.data() + 7 * H * D * 2, 0, 1, &one, B, H, D, 1, host[0].data(),
                     kvb, host[1].data(), kvb, ks, scb / 4, vs, scb / 4);
    for (int p = 0; p < 4; ++p) CHECK(to_host(ptr[p], size[p]) == host[p]);
    {
      // decode over the local FP8 pools == decode over a page-major FP8 arena
      // (one layer) holding block b's K and V planes as page b
      const uint64_t half8 = B * H * D, plane = B * H;
      std::vector<uint8_t> arena8(8 * 2 * half8);
      std::vector<float> sc8(8 * 2 * plane);
      for (int b = 0; b < 8; ++b) {
        std::memcpy(&arena8[(2 * b) * half8], host[0].data() + b * half8, half8);
        std::memcpy(&arena8[(2 * b + 1) * half8], host[1].data() + b * half8, half8);
        std::memcpy(&sc8[(2 * b) * plane], ks + b * plane, plane * 4);
        std::memcpy(&sc8[(2 * b + 1) * plane], vs + b * plane, plane * 4);
      }
      const int kvm = 4, batch = 3, max_blocks = 3;
      const std::vector<int32_t> local{5, 2, 7, 0, 3, -1, 6, 1, 4};
      std::vector<int32_t> paged(local);
      for (auto& id : paged) id = id < 0 ? -1 : 2 * id;
      const std::vector<int32_t> lens{40, 17, 48};
      uint8_t* da = to_device(arena8);
      float* dsc = to_device(sc8);
      int32_t* dtl = to_device(local);
      int32_t* dtp = to_device(paged);
      int32_t* dl = to_device(lens);
      const auto q = random_bf16(batch * kvm * H * D, 31);
      uint8_t* dq = to_device(q);
      uint8_t *o1 = nullptr, *o2 = nullptr, *ws = nullptr;
      const int32_t splits = 2;
      const uint64_t ws_bytes = pbe_paged_decode_workspace_bytes(batch, kvm * H, D, splits);
      HIP_OK(hipMalloc(&o1, q.size()));
      HIP_OK(hipMalloc(&o2, q.size()));
      HIP_OK(hipMalloc(&ws, ws_bytes));
      model::PagedKVDecodeRuntimeArgs a;
      a.batch_size = batch;
      a.head_num = kvm * H;
      a.head_size = D;
      a.kv_mul = kvm;
      a.max_blocks_per_seq = max_blocks;
      a.block_size = B;
      a.num_kv_heads = H;
      a.queries = dq;
      a.outputs = o1;
      a.block_tables = dtl;
      a.seq_lens = dl;
      a.workspace = ws;
      a.workspace_bytes = ws_bytes;
      a.splits = splits;
      CHECK(runtime.decode(pool, a));
      pbe_arena_view v8{};
      v8.base[0] = da;
      v8.bytes = v8.segment_bytes = arena8.size();
      v8.nseg = 1;
      const pbe_kv_shape shape{1, H, D, B};
      REQUIRE(pbe_paged_decode(&v8, PBE_KV_FP8_E4M3, dsc, sc8.size() * 4, &shape, 0, dq, o2, batch, kvm * H, dtp,
                               dl, max_blocks, splits, ws, ws_bytes, 0, stream) == PBE_OK);
      REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
      const auto got = to_host(o1, q.size());
      CHECK(got == to_host(o2, q.size()));
      CHECK(std::any_of(got.begin(), got.end(), [](uint8_t b) { return b != 0; }));
      for (void* d : {static_cast<void*>(da), static_cast<void*>(dsc), static_cast<void*>(dtl),
                      static_cast<void*>(dtp), static_cast<void*>(dl), static_cast<void*>(dq),
                      static_cast<void*>(o1), static_cast<void*>(o2), static_cast<void*>(ws)})
        HIP_OK(hipFree(d));
    }
    HIP_OK(hipFree(dK));
    HIP_OK(hipFree(dV));
    HIP_OK(hipFree(dS));
  }
  {
    // (3) a plain FP32 pool: FP32 input is written as is; BF16 input, which the
    // pool's element type does not match, is refused; the reader declines it.
    base::BlockAllocator f32(4, B, H, D, base::DataType::kDataTypeFp32, base::DeviceType::kDeviceHIP);
    const base::KVPoolView pool = f32.pool_view();
    const size_t kvb = pool.key_pool_bytes();
    CHECK_EQ(kvb, 4u * B * H * D * 4);
    std::vector<uint8_t> hk = random_bytes(kvb, 61), hv = random_bytes(kvb, 62);
    HIP_OK(hipMemcpy(pool.key_pool(), hk.data(), kvb, hipMemcpyHostToDevice));
    HIP_OK(hipMemcpy(pool.value_pool(), hv.data(), kvb, hipMemcpyHostToDevice));
    const int n = 5;
    const std::vector<int32_t> slots{17, 3, 63, -1, 40};
    const auto K = random_bytes(n * H * D * 4, 63), V = random_bytes(n * H * D * 4, 64);
    uint8_t* dK = to_device(K);
    uint8_t* dV = to_device(V);
    int32_t* dS = to_device(slots);
    REQUIRE(dK && dV && dS);
    runtime.scatter(dK, dV, base::DataType::kDataTypeFp32, pool, dS, B, H, D, n);
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    float none = 0.f;
    oracle_scatter()(K.data(), V.data(), 1, n, slots.data(), B, H, D, 0, hk.data(), kvb, hv.data(), kvb, &none, 0,
                     &none, 0);
    CHECK(to_host(pool.key_pool(), kvb) == hk);
    CHECK(to_host(pool.value_pool(), kvb) == hv);
    CHECK_THROWS_AS(runtime.scatter(dK, dV, base::DataType::kDataTypeBf16, pool, dS, B, H, D, n),
                    std::invalid_argument);
    model::PagedKVDecodeRuntimeArgs a;
    a.batch_size = 1;
    a.head_num = 2 * H;
    a.head_size = D;
    a.kv_mul = 2;
    a.max_blocks_per_seq = 1;
    a.block_size = B;
    a.num_kv_heads = H;
    a.queries = dK;
    a.outputs = dV;
    a.block_tables = dS;
    a.seq_lens = dS;
    a.workspace = dK;
    a.workspace_bytes = K.size();
    CHECK(!runtime.decode(pool, a));  // FP32 pages: not a reader dtype, nothing launched
    HIP_OK(hipFree(dK));
    HIP_OK(hipFree(dV));
    HIP_OK(hipFree(dS));
  }
  {
    // (4) decode_append over twin FP8 pools == scatter of the step's tokens
    // at their last positions, then decode: all four pools and the outputs.
    const int nblk = 12, kvm = 6, batch = 4, max_blocks = 4;
    base::BlockAllocator one(nblk, B, H, D, base::DataType::kDataTypeBf16, base::DeviceType::kDeviceHIP,
                             base::BlockStorageMode::kFp8E4M3PerTokenHead);
    base::BlockAllocator two(nblk, B, H, D, base::DataType::kDataTypeBf16, base::DeviceType::kDeviceHIP,
                             base::BlockStorageMode::kFp8E4M3PerTokenHead);
    const base::KVPoolView p1 = one.pool_view(), p2 = two.pool_view();
    const size_t kvb = p1.key_pool_bytes(), scb = p1.scale_pool_bytes();
    for (int p = 0; p < 4; ++p) {
      std::vector<uint8_t> h = random_bytes(p < 2 ? kvb : scb, 70 + p);
      if (p < 2) {
        for (auto& c : h) c = (c & 0x7f) == 0x7f ? 0 : c;  // no NaN codes
      } else {
        auto* f = reinterpret_cast<float*>(h.data());
        for (size_t i = 0; i < scb / 4; ++i) f[i] = 0.001f + 0.01f * (h[4 * i] / 255.f);
      }
      void* d1[4] = {p1.key_pool(), p1.value_pool(), p1.key_scale_pool(), p1.value_scale_pool()};
      void* d2[4] = {p2.key_pool(), p2.value_pool(), p2.key_scale_pool(), p2.value_scale_pool()};
      HIP_OK(hipMemcpy(d1[p], h.data(), h.size(), hipMemcpyHostToDevice));
      HIP_OK(hipMemcpy(d2[p], h.data(), h.size(), hipMemcpyHostToDevice));
    }
    const std::vector<int32_t> table{3, 7, 1, 10, 0, -1, -1, -1, 5, 9, 2, -1, 11, 4, 8, 6};
    const std::vector<int32_t> lens{64, 1, 33, 50};
    std::vector<int32_t> slots;
    for (int b = 0; b < batch; ++b) slots.push_back(table[b * max_blocks + (lens[b] - 1) / B] * B + (lens[b] - 1) % B);
    const auto K = random_bf16(batch * H * D, 81), V = random_bf16(batch * H * D, 82);
    const auto q = random_bf16(batch * kvm * H * D, 83);
    uint8_t* dK = to_device(K);
    uint8_t* dV = to_device(V);
    uint8_t* dq = to_device(q);
    int32_t* dS = to_device(slots);
    int32_t* dt = to_device(table);
    int32_t* dl = to_device(lens);
    REQUIRE(dK && dV && dq && dS && dt && dl);
    const int32_t splits = 2;
    const uint64_t ws_bytes = pbe_paged_decode_workspace_bytes(batch, kvm * H, D, splits);
    uint8_t *o1 = nullptr, *o2 = nullptr, *ws = nullptr;
    HIP_OK(hipMalloc(&o1, q.size()));
    HIP_OK(hipMalloc(&o2, q.size()));
    HIP_OK(hipMalloc(&ws, ws_bytes));
    model::PagedKVDecodeRuntimeArgs a;
    a.batch_size = batch;
    a.head_num = kvm * H;
    a.head_size = D;
    a.kv_mul = kvm;
    a.max_blocks_per_seq = max_blocks;
    a.block_size = B;
    a.num_kv_heads = H;
    a.queries = dq;
    a.outputs = o1;
    a.block_tables = dt;
    a.seq_lens = dl;
    a.workspace = ws;
    a.workspace_bytes = ws_bytes;
    a.splits = splits;
    runtime.scatter(dK, dV, base::DataType::kDataTypeBf16, p1, dS, B, H, D, batch);
    CHECK(runtime.decode(p1, a));
    a.outputs = o2;
    CHECK(runtime.decode_append(p2, a, dK, dV));
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    CHECK(to_host(p1.key_pool(), kvb) == to_host(p2.key_pool(), kvb));
    CHECK(to_host(p1.value_pool(), kvb) == to_host(p2.value_pool(), kvb));
    CHECK(to_host(p1.key_scale_pool(), scb) == to_host(p2.key_scale_pool(), scb));
    CHECK(to_host(p1.value_scale_pool(), scb) == to_host(p2.value_scale_pool(), scb));
    const auto got = to_host(o2, q.size());
    CHECK(got == to_host(o1, q.size()));
    CHECK(std::any_of(got.begin(), got.end(), [](uint8_t b) { return b != 0; }));
    CHECK_THROWS_AS(runtime.decode_append(p2, a, dK, nullptr), std::invalid_argument);
    for (void* d : {static_cast<void*>(dK), static_cast<void*>(dV), static_cast<void*>(dq), static_cast<void*>(dS),
                    static_cast<void*>(dt), static_cast<void*>(dl), static_cast<void*>(o1), static_cast<void*>(o2),
                    static_cast<void*>(ws)})
      HIP_OK(hipFree(d));
  }
  REQUIRE(pbe_stream_destroy(0, stream) == PBE_OK);
}

TEST_CASE("model runtime: a chunk's query tokens attend to its pages") {
  const int H = 2, D = 128, B = 16, nblk = 12, kvm = 6, batch = 3, max_blocks = 4, spare = 2;
  void* stream = nullptr;
  REQUIRE(pbe_stream_create(0, &stream) == PBE_OK);
  const model::HipPagedKVRuntime runtime(0, stream);
  const std::vector<int32_t> table{3, 7, 1, 10, 0, 6, -1, -1, 5, 9, 2, -1}, lens{64, 20, 33}, starts{0, 30, 31, 64};
  const int rows = starts[batch] + spare;
  const auto q = random_bf16(rows * kvm * H * D, 91);
  int32_t* dt = to_device(table);
  int32_t* dl = to_device(lens);
  int32_t* ds = to_device(starts);
  uint8_t* dq = to_device(q);
  const uint64_t ws_bytes = pbe_prompt_workspace_bytes(rows, batch, kvm * H, H, D);
  const int32_t splits = 2;
  const uint64_t decode_bytes = pbe_paged_decode_workspace_bytes(batch, kvm * H, D, splits);
  uint8_t *o1 = nullptr, *o2 = nullptr, *ws = nullptr;
  HIP_OK(hipMalloc(&o1, q.size()));
  HIP_OK(hipMalloc(&o2, q.size()));
  HIP_OK(hipMalloc(&ws, std::max(ws_bytes, decode_bytes)));
  REQUIRE(dt && dl && ds && dq);
  for (const bool fp8 : {false, true}) {
    base::BlockAllocator blocks(nblk, B, H, D, base::DataType::kDataTypeBf16, base::DeviceType::kDeviceHIP,
                                fp8 ? base::BlockStorageMode::kFp8E4M3PerTokenHead : base::BlockStorageMode::kPlain);
    const base::KVPoolView pool = blocks.pool_view();
    // every token's K and V, written by the runtime itself
    const auto K = random_bf16(nblk * B * H * D, 92), V = random_bf16(nblk * B * H * D, 93);
    std::vector<int32_t> slots(nblk * B);
    for (int i = 0; i < nblk * B; ++i) slots[i] = i;
    uint8_t* dK = to_device(K);
    uint8_t* dV = to_device(V);
    int32_t* dS = to_device(slots);
    REQUIRE(dK && dV && dS);
    runtime.scatter(dK, dV, base::DataType::kDataTypeBf16, pool, dS, B, H, D, nblk * B);
    HIP_OK(hipMemset(o1, 0x3f, q.size()));
    HIP_OK(hipMemset(o2, 0x3f, q.size()));
    model::PagedKVPrefillRuntimeArgs a;
    a.n_rows = rows;
    a.batch_size = batch;
    a.head_num = kvm * H;
    a.head_size = D;
    a.kv_mul = kvm;
    a.max_blocks_per_seq = max_blocks;
    a.block_size = B;
    a.num_kv_heads = H;
    a.queries = dq;
    a.outputs = o1;
    a.token_starts = ds;
    a.block_tables = dt;
    a.seq_lens = dl;
    a.workspace = ws;
    a.workspace_bytes = ws_bytes;
    CHECK(runtime.prefill(pool, a));
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    const auto got = to_host(o1, q.size());
    const size_t row = static_cast<size_t>(kvm) * H * D * 2;
    for (size_t i = starts[batch] * row; i < got.size(); ++i) REQUIRE(got[i] == 0x3f);  // rows of no sequence
    REQUIRE(pbe_paged_prompt_attention(pool.key_pool(), pool.value_pool(), pool.key_pool_bytes(),
                                       fp8 ? pool.key_scale_pool() : nullptr, fp8 ? pool.value_scale_pool() : nullptr,
                                       fp8 ? pool.scale_pool_bytes() : 0, fp8 ? PBE_KV_FP8_E4M3 : PBE_KV_BF16, H, D, dq,
                                       o2, rows, ds, batch, kvm * H, dt, dl, max_blocks, ws, ws_bytes, 0,
                                       stream) == PBE_OK);
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    CHECK(got == to_host(o2, q.size()));
    // A sequence's last row sees what a decode step sees. Of values below M each reader
    // is off by less than 2^-8 (its output's rounding) + 2^-8 (its weights') and a
    // little of M.
    std::vector<uint8_t> last;
    for (int b = 0; b < batch; ++b) last.insert(last.end(), q.begin() + (starts[b + 1] - 1) * row, q.begin() + starts[b + 1] * row);
    uint8_t* dlast = to_device(last);
    REQUIRE(dlast);
    model::PagedKVDecodeRuntimeArgs d;
    d.batch_size = batch;
    d.head_num = kvm * H;
    d.head_size = D;
    d.kv_mul = kvm;
    d.max_blocks_per_seq = max_blocks;
    d.block_size = B;
    d.num_kv_heads = H;
    d.queries = dlast;
    d.outputs = o2;
    d.block_tables = dt;
    d.seq_lens = dl;
    d.workspace = ws;
    d.workspace_bytes = decode_bytes;
    d.splits = splits;
    CHECK(runtime.decode(pool, d));
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    const auto one = to_host(o2, batch * row);
    auto value = [](const std::vector<uint8_t>& x, size_t i) {
      const uint32_t bits = (static_cast<uint32_t>(x[2 * i]) | static_cast<uint32_t>(x[2 * i + 1]) << 8) << 16;
      float f;
      std::memcpy(&f, &bits, 4);
      return f;
    };
    float most = 0.f, apart = 0.f;
    for (size_t i = 0; i < V.size() / 2; ++i) most = std::max(most, std::fabs(value(V, i)));
    for (int b = 0; b < batch; ++b)
      for (size_t i = 0; i < row / 2; ++i)
        apart = std::max(apart, std::fabs(value(one, b * row / 2 + i) - value(got, (starts[b + 1] - 1) * row / 2 + i)));
    CHECK(apart <= 2.f * (1.f / 128.f + 1.f / 4096.f) * most * (fp8 ? 1.0625f : 1.f));  // E4M3 values: 2^-4 more
    // no workspace: the same to within the order of sums, and in place
    a.workspace = nullptr;
    a.workspace_bytes = 0;
    a.queries = a.outputs = o1;
    HIP_OK(hipMemcpy(o1, q.data(), q.size(), hipMemcpyHostToDevice));
    CHECK(runtime.prefill(pool, a));
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    a.queries = dq;
    a.block_size = 32;
    CHECK(!runtime.prefill(pool, a));
    a.block_size = B;
    a.head_size = 96;
    CHECK(!runtime.prefill(pool, a));
    a.head_size = D;
    a.kv_mul = 5;
    CHECK_THROWS_AS(runtime.prefill(pool, a), std::invalid_argument);
    a.kv_mul = kvm;
    a.outputs = dq + 16;
    CHECK_THROWS_AS(runtime.prefill(pool, a), std::invalid_argument);
    a.outputs = nullptr;
    CHECK_THROWS_AS(runtime.prefill(pool, a), std::invalid_argument);
    for (void* x : {static_cast<void*>(dK), static_cast<void*>(dV), static_cast<void*>(dS), static_cast<void*>(dlast)}) HIP_OK(hipFree(x));
  }
  for (void* x : {static_cast<void*>(dt), static_cast<void*>(dl), static_cast<void*>(ds), static_cast<void*>(dq), static_cast<void*>(o1),
                  static_cast<void*>(o2), static_cast<void*>(ws)})
    HIP_OK(hipFree(x));
  REQUIRE(pbe_stream_destroy(0, stream) == PBE_OK);
}

TEST_CASE("model runtime: a long chunk without a workspace, over its queries") {
  const int H = 2, D = 128, B = 16, nblk = 70, kvm = 6, max_blocks = 66;
  void* stream = nullptr;
  REQUIRE(pbe_stream_create(0, &stream) == PBE_OK);
  const model::HipPagedKVRuntime runtime(0, stream);
  std::vector<int32_t> table(2 * max_blocks, -1);
  for (int i = 0; i < 63; ++i) table[i] = (i * 11) % nblk;  // 11 and 70 have no factor in common: blocks of their own
  for (int i = 0; i < 3; ++i) table[max_blocks + i] = ((63 + i) * 11) % nblk;
  const std::vector<int32_t> lens{1000, 40}, starts{0, 45, 85};
  const int rows = starts[2] + 1;
  const size_t row = static_cast<size_t>(kvm) * H * D * 2;
  const auto q = random_bf16(rows * kvm * H * D, 95);
  int32_t* dt = to_device(table);
  int32_t* dl = to_device(lens);
  int32_t* ds = to_device(starts);
  uint8_t* dq = to_device(q);
  const uint64_t ws_bytes = pbe_prompt_workspace_bytes(rows, 2, kvm * H, H, D);
  REQUIRE(ws_bytes > 0);
  uint8_t *out = nullptr, *ws = nullptr;
  HIP_OK(hipMalloc(&out, q.size()));
  HIP_OK(hipMalloc(&ws, ws_bytes));
  REQUIRE(dt && dl && ds && dq);
  auto value = [](const std::vector<uint8_t>& x, size_t i) {
    const uint32_t bits = (static_cast<uint32_t>(x[2 * i]) | static_cast<uint32_t>(x[2 * i + 1]) << 8) << 16;
    float f;
    std::memcpy(&f, &bits, 4);
    return f;
  };
  for (const bool fp8 : {false, true}) {
    base::BlockAllocator blocks(nblk, B, H, D, base::DataType::kDataTypeBf16, base::DeviceType::kDeviceHIP,
                                fp8 ? base::BlockStorageMode::kFp8E4M3PerTokenHead : base::BlockStorageMode::kPlain);
    const base::KVPoolView pool = blocks.pool_view();
    const auto K = random_bf16(nblk * B * H * D, 96), V = random_bf16(nblk * B * H * D, 97);
    std::vector<int32_t> slots(nblk * B);
    for (int i = 0; i < nblk * B; ++i) slots[i] = i;
    uint8_t* dK = to_device(K);
    uint8_t* dV = to_device(V);
    int32_t* dS = to_device(slots);
    REQUIRE(dK && dV && dS);
    runtime.scatter(dK, dV, base::DataType::kDataTypeBf16, pool, dS, B, H, D, nblk * B);
    HIP_OK(hipMemset(out, 0x3f, q.size()));
    model::PagedKVPrefillRuntimeArgs a;
    a.n_rows = rows;
    a.batch_size = 2;
    a.head_num = kvm * H;
    a.head_size = D;
    a.kv_mul = kvm;
    a.max_blocks_per_seq = max_blocks;
    a.block_size = B;
    a.num_kv_heads = H;
    a.queries = dq;
    a.outputs = out;
    a.token_starts = ds;
    a.block_tables = dt;
    a.seq_lens = dl;
    a.workspace = ws;
    a.workspace_bytes = ws_bytes;
    CHECK(runtime.prefill(pool, a));
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    const auto in_parts = to_host(out, q.size());
    a.workspace = nullptr;
    a.workspace_bytes = 0;
    a.queries = out;
    HIP_OK(hipMemcpy(out, q.data(), q.size(), hipMemcpyHostToDevice));
    CHECK(runtime.prefill(pool, a));
    REQUIRE(pbe_stream_synchronize(0, stream) == PBE_OK);
    const auto whole = to_host(out, q.size());
    // Of values below M either is off by less than 2^-8 M by its output's rounding, 2^-8
    // (1 + 2^-7) M by its weights', and 2^-12 M by FP32's.
    float most = 0.f, apart = 0.f;
    for (size_t i = 0; i < V.size() / 2; ++i) most = std::max(most, std::fabs(value(V, i)));
    bool numbers = true;
    for (size_t i = 0; i < starts[2] * row / 2; ++i) {
      numbers &= std::isfinite(value(whole, i)) && std::isfinite(value(in_parts, i));
      apart = std::max(apart, std::fabs(value(whole, i) - value(in_parts, i)));
    }
    CHECK(numbers);
    CHECK(apart <= 2.f * (1.f / 128.f + 1.f / 2048.f) * most * (fp8 ? 1.0625f : 1.f));  // E4M3 values: 2^-4 more
    bool kept = true;  // the row behind the last sequence: what was there
    for (size_t i = starts[2] * row; i < q.size(); ++i) kept &= whole[i] == q[i] && in_parts[i] == 0x3f;
    CHECK(kept);
    for (void* x : {static_cast<void*>(dK), static_cast<void*>(dV), static_cast<void*>(dS)}) HIP_OK(hipFree(x));
  }
  for (void* x : {static_cast<void*>(dt), static_cast<void*>(dl), static_cast<void*>(ds), static_cast<void*>(dq), static_cast<void*>(out), static_cast<void*>(ws)})
    HIP_OK(hipFree(x));
  REQUIRE(pbe_stream_destroy(0, stream) == PBE_OK);
}

MINITEST_MAIN()
