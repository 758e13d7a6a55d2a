// The launch recorder, which also writes down what kernels are allowed of LDS, call by call.
#define hipFuncSetAttribute attribute_not_written_down
#include "launch_recorder.cpp"
#undef hipFuncSetAttribute

namespace {
struct Limit {
    std::string name;
    int attribute, value;
};
std::vector<Limit> &limits()
{
    static std::vector<Limit> v;
    return v;
}
} // namespace

extern "C" {
int hipFuncSetAttribute(const void *f, int attribute, int value)
{
    limits().push_back(Limit{ names()[f], attribute, value });
    return 0;
}
int limit_count() { return (int)limits().size(); }
const char *limit_name(int i) { return limits()[i].name.c_str(); }
int limit_value(int i) { return limits()[i].value; }
}
