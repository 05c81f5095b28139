// host_errors.h -- how the host extension's parts raise Python exceptions, and
// the parts that _suika_host is made of.
#ifndef SUIKA_HOST_ERRORS_H
#define SUIKA_HOST_ERRORS_H

#include <pybind11/pybind11.h>

#include <string>

#include "suika_reshard.h"

namespace suika_host {

namespace py = pybind11;

inline PyObject* lib_exception(const char* name) {
  py::object mod = py::module_::import("suika_amd._lib");
  py::object cls = mod.attr(name);
  return cls.release().ptr();   // a new reference, kept for the process
}

inline const char* status_name(int rc) {
  switch (rc) {
    case SR_OK: return "SR_OK";
    case SR_EINVAL: return "SR_EINVAL";
    case SR_EBOUNDS: return "SR_EBOUNDS";
    case SR_EALIGN: return "SR_EALIGN";
    case SR_EOVERLAP: return "SR_EOVERLAP";
    case SR_EHIP: return "SR_EHIP";
    case SR_ENOMEM: return "SR_ENOMEM";
    case SR_EDTYPE: return "SR_EDTYPE";
    default: return nullptr;
  }
}

// "<what>: <status>: <message>", as suika_amd._lib.check words it:
// suika_amd._lib.PlanError, or ReshardError for device and memory failures.
[[noreturn]] inline void raise_status(int rc, const char* what, const std::string& msg) {
  static PyObject* plan_error = lib_exception("PlanError");
  static PyObject* reshard_error = lib_exception("ReshardError");
  const char* name = status_name(rc);
  const std::string text = std::string(what) + ": " + (name ? name : std::to_string(rc)) + ": " + msg;
  PyErr_SetString(rc == SR_EHIP || rc == SR_ENOMEM ? reshard_error : plan_error, text.c_str());
  throw py::error_already_set();
}

inline void check(int rc, const char* what) {
  if (rc != SR_OK) raise_status(rc, what, sr_last_error());
}

// A refused argument.
[[noreturn]] inline void plan_error(const std::string& msg) {
  static PyObject* cls = lib_exception("PlanError");
  PyErr_SetString(cls, msg.c_str());
  throw py::error_already_set();
}

// The training-step operators (step_bind.cpp).
void bind_step(py::module_& m);

}  // namespace suika_host

#endif  // SUIKA_HOST_ERRORS_H
