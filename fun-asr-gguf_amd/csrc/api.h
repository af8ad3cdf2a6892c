// The try / catch frame of every C entry point: a failure becomes a status code and a message (fa_last_error), and no
// exception leaves the library.
#pragma once
#include <exception>
#include "common.h"
#include "funasr_hip.h"

#define FA_API_BEGIN try {
#define FA_API_END                 \
  }                                \
  catch (fa::hip_failure&) {       \
    return FA_ERR_HIP;             \
  }                                \
  catch (fa::arg_failure&) {       \
    return FA_ERR_ARG;             \
  }                                \
  catch (std::exception & ex) {    \
    fa::set_error(ex.what());      \
    return FA_ERR_STATE;           \
  }                                \
  return FA_OK;
