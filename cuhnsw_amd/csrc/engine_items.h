// The vectors of an index as a table: rows by item, searches from items, all rows in 4 bits (engine.hip calls these with the
// engine's lock held).
//
// Items are named as a search names them: by label on an index that came from a file, else by row number.
#pragma once
#include "engine.h"
#include "rows.h"

namespace cuhnsw_amd {

class Items {
 public:
  // the index was replaced
  void forget() { label_order_.clear(); }

  void labels(Engine& g, int num_rows, long long* out) {
    same_index(g.host.N, num_rows, "rows");
    need_vectors(g, "get_labels");
    want(out, "get_labels: null argument");
    if (!g.host.labelled) {
      for (int i = 0; i < g.host.N; ++i) out[i] = i;
      return;
    }
    HIP_CHECK(hipMemcpyAsync(out, g.d_labels.p, (size_t)g.host.N * 8, hipMemcpyDeviceToHost, g.stream));
    HIP_CHECK(hipStreamSynchronize(g.stream));
  }

  void get(Engine& g, const int* items, int n, int num_dims, float scale, float* out) {
    same_index(g.host.D, num_dims, "elements a vector");
    need_vectors(g, "get_items");
    if (n <= 0) return;
    want(items && out, "get_items: null argument");
    look_up(g, items, n, scale);
    HIP_CHECK(hipMemcpyAsync(out, g.d_q.p, (size_t)n * g.host.D * 4, hipMemcpyDeviceToHost, g.stream));
    HIP_CHECK(hipStreamSynchronize(g.stream));
  }

  void search(Engine& g, const int* items, int n, float scale, int k, int ef, int* nns, float* dists, int* found) {
    need_vectors(g, "search_items");
    if (n <= 0) return;
    want(items && nns && dists && found, "search_items: null argument");
    want(k > 0, "search_items: topk must be positive");
    look_up(g, items, n, scale);
    g.d_nns.reserve((size_t)n * k);
    g.d_dist.reserve((size_t)n * k);
    g.d_found.reserve((size_t)n);
    g.search_device(g.d_q.p, n, k, ef, g.d_nns.p, g.d_dist.p, g.d_found.p, nullptr, nullptr);
    HIP_CHECK(hipMemcpyAsync(nns, g.d_nns.p, (size_t)n * k * 4, hipMemcpyDeviceToHost, g.stream));
    HIP_CHECK(hipMemcpyAsync(dists, g.d_dist.p, (size_t)n * k * 4, hipMemcpyDeviceToHost, g.stream));
    HIP_CHECK(hipMemcpyAsync(found, g.d_found.p, (size_t)n * 4, hipMemcpyDeviceToHost, g.stream));
    HIP_CHECK(hipStreamSynchronize(g.stream));
  }

  // On the caller's stream, and waited for: the vectors may be replaced by the next call.
  void pack(Engine& g, int num_rows, int num_dims, int group, void* codes, void* scales, void* offsets, int scale_type, hipStream_t stream) {
    same_index(g.host.N, num_rows, "rows");
    same_index(g.host.D, num_dims, "elements a vector");
    need_vectors(g, "pack_items");
    want(group == 32 || group == 64 || group == 128, "pack_items: the group is 32, 64 or 128 elements");
    want(scale_type == TYPE_F16 || scale_type == TYPE_BF16, "pack_items: scales are float16 or bfloat16");
    want(codes && scales && (reinterpret_cast<uintptr_t>(codes) & 15) == 0, "pack_items: codes and scales are wanted, the codes aligned to 16 bytes");
    int device = -1;
    HIP_CHECK(hipGetDevice(&device));
    want(device == g.device_ordinal, "pack_items: the index is on another device than the current one");
    launch_pack({g.d_vectors.p, g.storage_half ? TYPE_F16 : TYPE_F32, g.Dp, g.host.N, g.host.D, group, static_cast<unsigned char*>(codes), scales,
                 offsets, scale_type}, stream);
    HIP_CHECK(hipStreamSynchronize(stream));
  }

 private:
  // Another thread's call may have put another index in the place of the one that the caller made room for.
  static void same_index(int has, int expected, const char* what) {
    if (has != expected)
      throw std::runtime_error("the index was replaced meanwhile: " + std::to_string(has) + " " + what + ", not " + std::to_string(expected));
  }
  static void need_vectors(const Engine& g, const char* what) {
    g.need_device();
    if (!g.have_data) throw std::runtime_error(std::string(what) + ": no vectors (call set_data or load_index first)");
  }

  // the items' rows, times scale, into the engine's buffer for queries
  void look_up(Engine& g, const int* items, int n, float scale) {
    std::vector<int> rows(items, items + n);
    if (g.host.labelled && label_order_.empty()) {
      std::vector<long long> labels_of((size_t)g.host.N);
      labels(g, g.host.N, labels_of.data());
      std::vector<std::pair<uint64_t, int>> order((size_t)g.host.N);
      for (int i = 0; i < g.host.N; ++i) order[(size_t)i] = {(uint64_t)labels_of[(size_t)i], i};
      std::sort(order.begin(), order.end());
      label_order_.swap(order);
    }
    for (int& r : rows) {
      if (g.host.labelled) {
        const auto at = std::lower_bound(label_order_.begin(), label_order_.end(), std::make_pair((uint64_t)std::max(r, 0), 0));
        if (r < 0 || at == label_order_.end() || at->first != (uint64_t)r) throw std::runtime_error("no item has the label " + std::to_string(r));
        r = at->second;
      } else if (r < 0 || r >= g.host.N) {
        throw std::runtime_error("item " + std::to_string(r) + " is outside the index");
      }
    }
    g.d_q.reserve((size_t)n * g.host.D);
    rows_there_.reserve((size_t)n);
    HIP_CHECK(hipMemcpyAsync(rows_there_.p, rows.data(), (size_t)n * 4, hipMemcpyHostToDevice, g.stream));
    launch_lookup({g.d_vectors.p, g.storage_half ? TYPE_F16 : TYPE_F32, g.host.N, g.Dp, g.host.D, rows_there_.p, 0, n, scale, g.d_q.p, TYPE_F32},
                  g.stream);
    HIP_CHECK(hipStreamSynchronize(g.stream));  // (a search goes on with the rows on two streams)
  }

  std::vector<std::pair<uint64_t, int>> label_order_;  // (label, row), ascending; made when first asked for
  DevBuf<int> rows_there_;
};

}  // namespace cuhnsw_amd
