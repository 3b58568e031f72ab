// what a kernel file takes from csrc/dsp_capi.cpp, for an interpreter library of that file alone
#include <string>
static std::string g_error;
extern "C" void dsp_set_error_(const char* m) { g_error = m ? m : ""; }
extern "C" const char* dsp_last_error(void) { return g_error.c_str(); }
