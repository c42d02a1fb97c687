// tree_plan.cuh -- the plan object behind KvlMlaTreePlan.
#pragma once
#include "kvl/mla_cuda.h"
#include "tree_attend.cuh"

struct KvlMlaTreePlan {
  int device = 0;
  int nh = 0, R = 0;
  kvl::TreeHostPlan host;
  void *d_meta = nullptr;  // error word, then the arrays below
  void *d_work = nullptr;  // partial outputs and lse values
  size_t off_items = 0, off_merge = 0, off_row0 = 0, off_len = 0, off_tree = 0, off_first = 0,
         off_seq = 0, off_rows = 0;
};
