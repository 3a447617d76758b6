// Groups and handles of expert parallelism as the host code keeps them (nccl_ep.cc makes and frees them).
#pragma once
#include "nccl_ep.h"

#include <atomic>
#include <initializer_list>

#include "../comm/device_plane.h"
#include "ep_kernels.cuh"

using b200::EpArgs;
using b200::SymWindow;

struct ncclEpGroup {
  ncclComm* comm = nullptr;
  ncclEpGroupConfig_t cfg;
  int n = 1, E = 0, El = 0, H = 0, maxTokens = 0, K = 0;
  size_t slotBytes = 0, zoneBytes = 0, combZoneBytes = 0;
  char* recvZone = nullptr;           // 2 zones (epoch parity)
  SymWindow* recvWin = nullptr;
  char* ctl = nullptr;                // counts [2][El][n] u64, combine flags [n] u64
  SymWindow* ctlWin = nullptr;
  char* combZone = nullptr;           // 2 zones, allocated with the first handle (needs top-k)
  SymWindow* combWin = nullptr;
  uint32_t* state = nullptr;
  uint32_t* mask = nullptr;           // [n] device words: non-zero = that rank is left out of dispatch / combine
  int smCount = 0;
  int lastError = 0;
  std::atomic<int> expertPairs{-1};   // clusters of the experts' products on CTA pairs that can be resident at once (-1: not asked yet)
  int layoutClass = 0;                // 0 none yet, 1 expert-major, 2 per-rank (rank-major / flat)
};

struct ncclEpHandle {
  ncclEpGroup* g = nullptr;
  ncclEpLayout_t layout;
  int K = 0, T = 0;
  int outSlots = 0;                   // flat layout: rows of the last dispatch's outputs
  const int64_t* topkIdx = nullptr;
  const float* topkW = nullptr;
  // routing of the last dispatch that was carried out (the two above may be those of one that was refused, or not made yet); null: none, or
  // its rows were given up half-way
  const int64_t* sentIdx = nullptr;
  int sentT = 0;
  int2* srcInfo = nullptr;
  int* rowOf = nullptr;               // one-rank groups, expert-major: where (token, k) went
  int* expertCount = nullptr;
  ncclEpAllocConfig_t alloc = {};     // the group's hooks, kept here so that a handle can outlive its group's record
  // a send_only call leaves its receiving half to ncclEpComplete
  int pending = 0;                    // 0 nothing, 1 dispatch, 2 combine
  EpArgs pendingArgs;
  int pendingCtas = 0;
  size_t pendingSmem = 0;
  void* pendingCounters = nullptr;    // layout_info->expert_counters of the pending dispatch
};

// Memory of a call, to see whether outputs share any with inputs (null: none).
struct Span {
  const void* data;
  size_t bytes;
};
inline bool overlap(std::initializer_list<Span> outputs, std::initializer_list<Span> inputs) {
  for (const Span& o : outputs)
    for (const Span& i : inputs)
      if (o.data && i.data && (const char*)o.data < (const char*)i.data + i.bytes && (const char*)i.data < (const char*)o.data + o.bytes) return true;
  return false;
}
