// Copies between the slots of caches and states: for every tensor, slot dst = slot src, whole or its leading positions (a fork of a live sequence, the move of one).
//
// Bound: bytes.  Copies of one source are a group: a thread keeps what it read and writes it to every destination of the group, so the source is read once.
// A CTA takes 16 KB of one tensor's slot for one group; all tensors of a model go in as few launches as the parameter space takes, 128 tensors a launch, instead of one each.
// 15 copies of a request of 50 MB, 805 MB with the one read of it: 132 us (6.1 TB/s); six requests moved, 670 MB: 100 us (6.7 TB/s).
#include "common.cuh"

namespace b200 {

namespace {

constexpr int kSlThreads = 256, kSlBytes = 16384;
// what a launch takes at most: tensors, groups, destinations
template <int T, int G, int D>
struct SlotLaunch {
  static constexpr int kTensors = T, kGroups = G, kDst = D;
  unsigned char* base[T];
  int64_t slot_bytes[T], row_bytes[T];
  int64_t rows[G];               // leading positions, < 0: the whole slot
  int first_unit[T + 1];         // in units of 16 KB of every group
  int src[G], dst_first[G + 1], dst[D];
  int tensors, groups;
};

template <typename W>
__device__ __forceinline__ void copy_units(const unsigned char* src, unsigned char* base, int64_t slot_bytes, const int* dst, int n_dst, int64_t off, int64_t end) {
  constexpr int U = 4;
  const int64_t last = end / (int64_t)sizeof(W), first = off / (int64_t)sizeof(W), stop = min(last, (off + kSlBytes) / (int64_t)sizeof(W));
  for (int64_t i0 = first + threadIdx.x; i0 < stop; i0 += U * kSlThreads) {
    W v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * kSlThreads < stop) v[u] = reinterpret_cast<const W*>(src)[i0 + u * kSlThreads];
    for (int d = 0; d < n_dst; ++d) {
      W* const to = reinterpret_cast<W*>(base + (int64_t)dst[d] * slot_bytes);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * kSlThreads < stop) to[i0 + u * kSlThreads] = v[u];
    }
  }
  if (off + kSlBytes >= end) {   // the bytes behind the last whole unit
    const int64_t i = last * (int64_t)sizeof(W) + threadIdx.x;
    if (i < end)
      for (int d = 0; d < n_dst; ++d) base[(int64_t)dst[d] * slot_bytes + i] = src[i];
  }
}

template <typename L>
__global__ void __launch_bounds__(kSlThreads) copy_slots_kernel(const __grid_constant__ L p) {
  griddep_launch();
  griddep_wait();
  const int g = blockIdx.x % p.groups, unit = blockIdx.x / p.groups;
  int lo = 0, hi = p.tensors;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (p.first_unit[mid] <= unit) lo = mid; else hi = mid;
  }
  const int64_t slot = p.slot_bytes[lo], n = p.rows[g] < 0 ? slot : p.rows[g] * p.row_bytes[lo], off = (int64_t)(unit - p.first_unit[lo]) * kSlBytes;
  if (off >= n) return;
  unsigned char* const base = p.base[lo];
  const unsigned char* const src = base + (int64_t)p.src[g] * slot;
  const int* const dst = p.dst + p.dst_first[g];
  const int n_dst = p.dst_first[g + 1] - p.dst_first[g];
  const uintptr_t a = reinterpret_cast<uintptr_t>(base) | (uintptr_t)slot;
  if ((a & 15) == 0) copy_units<uint4>(src, base, slot, dst, n_dst, off, n);
  else if ((a & 3) == 0) copy_units<uint32_t>(src, base, slot, dst, n_dst, off, n);
  else if ((a & 1) == 0) copy_units<uint16_t>(src, base, slot, dst, n_dst, off, n);
  else copy_units<unsigned char>(src, base, slot, dst, n_dst, off, n);
}

template <typename L>
int launch_copies(const b200_slot_tensor* tensors, int n_tensors, const b200_slot_copy* copies, int n_copies, cudaStream_t stream) {
  L p;
  // groups: neighbouring copies of one source and length
  for (int c0 = 0; c0 < n_copies;) {
    p.groups = 0;
    p.dst_first[0] = 0;
    int64_t most = 0;      // positions of the longest group, < 0: whole slots
    bool whole = false;
    int c = c0, n_dst = 0;
    while (c < n_copies && n_dst < L::kDst) {
      const bool more = p.groups > 0 && copies[c].src == p.src[p.groups - 1] && copies[c].rows == p.rows[p.groups - 1];
      if (!more) {
        if (p.groups == L::kGroups) break;
        p.src[p.groups] = copies[c].src;
        p.rows[p.groups] = copies[c].rows;
        ++p.groups;
      }
      p.dst[n_dst++] = copies[c].dst;
      p.dst_first[p.groups] = n_dst;
      whole = whole || copies[c].rows < 0;
      most = copies[c].rows > most ? copies[c].rows : most;
      ++c;
    }
    for (int t0 = 0; t0 < n_tensors; t0 += L::kTensors) {
      p.tensors = n_tensors - t0 < L::kTensors ? n_tensors - t0 : L::kTensors;
      int64_t units = 0;
      for (int t = 0; t < p.tensors; ++t) {
        const b200_slot_tensor& x = tensors[t0 + t];
        p.base[t] = (unsigned char*)x.base;
        p.row_bytes[t] = x.row_bytes;
        p.slot_bytes[t] = x.row_bytes * x.rows;
        p.first_unit[t] = (int)units;
        const int64_t n = whole ? p.slot_bytes[t] : most * x.row_bytes;
        units += (n + kSlBytes - 1) / kSlBytes;
        B200_CHECK_ARG(units * p.groups < 0x7fffffff, "b200_copy_slots: too much at once");
      }
      p.first_unit[p.tensors] = (int)units;
      if (units) B200_CUDA(launch(copy_slots_kernel<L>, dim3((unsigned)(units * p.groups)), dim3(kSlThreads), 0, stream, p));
    }
    c0 = c;
  }
  return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_copy_slots(const b200_slot_tensor* tensors, int n_tensors, int slots, const b200_slot_copy* copies, int n_copies, b200_stream_t stream) {
  B200_CHECK_ARG(n_tensors >= 0 && n_copies >= 0 && (tensors || !n_tensors) && (copies || !n_copies), "b200_copy_slots: null argument");
  for (int t = 0; t < n_tensors; ++t)
    B200_CHECK_ARG(tensors[t].base && tensors[t].rows > 0 && tensors[t].row_bytes > 0, "b200_copy_slots: tensor %d is empty", t);
  for (int i = 0; i < n_copies; ++i) {
    const b200_slot_copy& c = copies[i];
    B200_CHECK_ARG(c.src >= 0 && c.src < slots && c.dst >= 0 && c.dst < slots, "b200_copy_slots: copy %d from slot %d to %d of %d", i, c.src, c.dst, slots);
    for (int t = 0; t < n_tensors && c.rows >= 0; ++t)
      B200_CHECK_ARG(c.rows <= tensors[t].rows, "b200_copy_slots: copy %d of %lld positions, tensor %d has %lld", i, (long long)c.rows, t, (long long)tensors[t].rows);
    for (int j = 0; j < n_copies; ++j) {
      B200_CHECK_ARG(c.dst != copies[j].src, "b200_copy_slots: slot %d is written by one copy and read by another", c.dst);
      B200_CHECK_ARG(j >= i || c.dst != copies[j].dst, "b200_copy_slots: slot %d is written twice", c.dst);
    }
  }
  if (!n_tensors || !n_copies) return B200_OK;
  // (a launch hands over its tables, 1 KB or 6 KB: a call for two tensors takes 6.6 and 7.0 us of the host)
  if (n_tensors <= 32 && n_copies <= 8) return launch_copies<SlotLaunch<32, 8, 8>>(tensors, n_tensors, copies, n_copies, (cudaStream_t)stream);
  return launch_copies<SlotLaunch<128, 64, 256>>(tensors, n_tensors, copies, n_copies, (cudaStream_t)stream);
}
