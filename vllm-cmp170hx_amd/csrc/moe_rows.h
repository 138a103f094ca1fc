// Row lists of a routed call: its slots grouped by expert without padding and
// cut into tasks, in two launches (count, fill).  Shared by the fused MoE paths
// that run on them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace moe {

// The slots come grouped by expert, in any order inside an expert (a row's sums
// depend on nothing but the row), cut into tasks {expert, first row, rows, 0},
// each expert's tasks of even height in whole 16-row blocks.
constexpr int kRowsPartThreads = 256;
constexpr int kRowsPartSlots = 8;
constexpr int kRowsPart = kRowsPartThreads * kRowsPartSlots;  // slots a workgroup counts
constexpr int kRowsMaxExperts = 1024;

// int32 offsets of the row lists' table: [tasks, 0, 0, 0], the tasks, the
// sorted slots, then each slot's place in its part (expert << 16 | place, or
// -1) and the parts' histograms.
struct RowsLayout {
  int64_t slots, experts, max_tasks;
  __host__ __device__ int64_t parts() const { return (slots + kRowsPart - 1) / kRowsPart; }
  __host__ __device__ int64_t tasks() const { return 4; }
  __host__ __device__ int64_t sorted() const { return 4 + 4 * max_tasks; }
  __host__ __device__ int64_t packed() const { return sorted() + (slots + 3) / 4 * 4; }
  __host__ __device__ int64_t hist() const { return packed() + (slots + 3) / 4 * 4; }
  __host__ __device__ int64_t total() const { return hist() + parts() * experts; }
};

// One part (workgroup `part`) of the count: the experts of its slots, as
// expert_of(slot) gives them (-1: left out), each slot's place among the part's
// rows of its expert, and the part's histogram.  part_count: `experts` ints of LDS.
template <typename ExpertOf>
__device__ __forceinline__ void rows_count_part(const ExpertOf& expert_of, const RowsLayout& lay, int32_t* table,
                                                int part, int* part_count) {
  const int experts = int(lay.experts);
  for (int e = threadIdx.x; e < experts; e += kRowsPartThreads) part_count[e] = 0;
  __syncthreads();
  const int64_t s0 = int64_t(part) * kRowsPart + threadIdx.x;
  int e[kRowsPartSlots];
#pragma unroll
  for (int u = 0; u < kRowsPartSlots; ++u) {
    const int64_t slot = s0 + u * kRowsPartThreads;
    e[u] = slot < lay.slots ? expert_of(slot) : -1;
  }
#pragma unroll
  for (int u = 0; u < kRowsPartSlots; ++u) {
    const int64_t slot = s0 + u * kRowsPartThreads;
    const int v = e[u] >= 0 ? (e[u] << 16) | atomicAdd(&part_count[e[u]], 1) : -1;
    if (slot < lay.slots) table[lay.packed() + slot] = v;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < experts; x += kRowsPartThreads) {
    table[lay.hist() + int64_t(part) * experts + x] = part_count[x];
  }
}

// Tasks of an expert of c rows, and the rows of each but the last.
__device__ __forceinline__ int rows_tasks(int c, int task_rows) { return (c + task_rows - 1) / task_rows; }
__device__ __forceinline__ int rows_height(int c, int tasks) {
  return tasks > 0 ? ((c + tasks - 1) / tasks + 15) / 16 * 16 : 16;
}

// One part (workgroup `part`) of the fill, first: `experts` ints of LDS (where
// this part's rows of the expert begin).  Every expert's first row (a scan of the summed
// histograms, the same in each workgroup) plus the rows of the parts before
// this one place the part's slots; workgroup 0 also writes the tasks.  Experts
// e0 .. e1 - 1 (a contiguous run) belong to one thread.
__device__ __forceinline__ void rows_fill_part(const RowsLayout& lay, int32_t* table, int task_rows, int part, int* first) {
  __shared__ int wave_rows[kRowsPartThreads / 64], wave_tasks[kRowsPartThreads / 64];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int experts = int(lay.experts);
  const int parts = int(lay.parts());
  const int per = (experts + kRowsPartThreads - 1) / kRowsPartThreads;
  constexpr int kPer = kRowsMaxExperts / kRowsPartThreads;
  const int e0 = tid * per;
  int total[kPer], before[kPer];
  int rows = 0, tasks = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    total[i] = before[i] = 0;
    const int e = e0 + i;
    if (i < per && e < experts) {
      for (int p0 = 0; p0 < parts; p0 += 8) {
        int n[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          n[u] = p0 + u < parts ? table[lay.hist() + int64_t(p0 + u) * experts + e] : 0;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          total[i] += n[u];
          if (p0 + u < part) before[i] += n[u];
        }
      }
      rows += total[i];
      const int h = rows_height(total[i], rows_tasks(total[i], task_rows));
      tasks += rows_tasks(total[i], h);
    }
  }
  int irows = rows, itasks = tasks;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int r = __shfl_up(irows, d), t = __shfl_up(itasks, d);
    if (lane >= d) {
      irows += r;
      itasks += t;
    }
  }
  if (lane == 63) {
    wave_rows[wave] = irows;
    wave_tasks[wave] = itasks;
  }
  __syncthreads();
  int row = irows - rows, task = itasks - tasks;
  for (int w = 0; w < wave; ++w) {
    row += wave_rows[w];
    task += wave_tasks[w];
  }
  if (part == 0 && tid == kRowsPartThreads - 1) table[0] = task + tasks;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = e0 + i;
    if (i < per && e < experts) {
      first[e] = row + before[i];
      if (part == 0) {
        const int h = rows_height(total[i], rows_tasks(total[i], task_rows));
        for (int r = 0; r < total[i]; r += h) {
          reinterpret_cast<int4*>(table + lay.tasks())[task++] = make_int4(e, row + r, min(h, total[i] - r), 0);
        }
      }
      row += total[i];
    }
  }
  __syncthreads();
  const int64_t s0 = int64_t(part) * kRowsPart + tid;
  int v[kRowsPartSlots];
#pragma unroll
  for (int u = 0; u < kRowsPartSlots; ++u) {
    const int64_t slot = s0 + u * kRowsPartThreads;
    v[u] = slot < lay.slots ? table[lay.packed() + slot] : -1;
  }
#pragma unroll
  for (int u = 0; u < kRowsPartSlots; ++u) {
    if (v[u] >= 0) table[lay.sorted() + first[v[u] >> 16] + (v[u] & 0xffff)] = int(s0 + u * kRowsPartThreads);
  }
}

}  // namespace moe
