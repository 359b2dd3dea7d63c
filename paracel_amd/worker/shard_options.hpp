// How a worker keeps and trains on its shard beyond what the reference's cfg files say: optional
// keys "storage" ("f64", the default, or "mxfp4": the training shard is held in 4 bits,
// plr_pack_data), "dropout" (the rate, default 0; needs "mxfp4") and "dropout_seed".
#pragma once

#include <errno.h>
#include <math.h>
#include <stdint.h>
#include <stdlib.h>

#include <map>
#include <stdexcept>
#include <string>

#include "../../include/plr.h"

namespace plr_ps {

struct shard_options {
  bool packed = false;
  double dropout = 0.;
  uint64_t seed = 0;

  void set(const std::string& key, const std::string& v) {
    if (key == "storage") {
      if (v != "f64" && v != "mxfp4") throw std::invalid_argument("storage must be f64 or mxfp4");
      packed = v == "mxfp4";
    } else if (key == "dropout") {
      char* end = nullptr;
      dropout = strtod(v.c_str(), &end);
      if (v.empty() || *end || !(dropout >= 0. && rint(dropout * 65536.) <= 65535.))  // as plr_set_dropout
        throw std::invalid_argument("dropout must be a rate of at least 0 and at most 65535/65536");
    } else if (key == "dropout_seed") {
      char* end = nullptr;
      errno = 0;
      seed = strtoull(v.c_str(), &end, 0);
      if (v.empty() || v.find('-') != std::string::npos || *end || errno == ERANGE)
        throw std::invalid_argument("dropout_seed must be a whole number from 0 to 2^64 - 1");
    }
  }
  static shard_options from(const std::map<std::string, std::string>& kv) {
    shard_options o;
    for (const char* k : {"storage", "dropout", "dropout_seed"})
      if (kv.count(k)) o.set(k, kv.at(k));
    o.check();
    return o;
  }
  void check() const {
    if (dropout > 0. && !packed) throw std::invalid_argument("dropout needs storage mxfp4");
  }
  // The training shard has become resident.
  int resident(plr_ctx* gpu) const { return packed ? plr_pack_data(gpu) : (int)PLR_OK; }
  // Before round rd: a new mask each round; a worker's rows are rows worker_id * 2^40 + i of the
  // whole, so that no two workers drop alike.
  int round(plr_ctx* gpu, int worker_id, int rd) const {
    if (!(dropout > 0.)) return PLR_OK;
    plr_dropout d;
    d.rate = dropout;
    d.seed = seed;
    d.row0 = (int64_t)worker_id << 40;
    d.step = (uint32_t)rd;
    return plr_set_dropout(gpu, &d);
  }
};

}  // namespace plr_ps
