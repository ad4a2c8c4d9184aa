// The 4-bit cache's and the verification's entry points with their arguments as
// one array of 64-bit words: a foreign-function interface that converts
// arguments one by one (ctypes: 2.2 us for 17) passes one pointer instead
// (0.7 us, packing included).
#include <cstring>

#include "common.cuh"

namespace {

template <typename T>
T* at(int64_t word) {
    return reinterpret_cast<T*>(static_cast<uintptr_t>(word));
}

float float_of(int64_t word) {
    float f;
    const uint32_t low = static_cast<uint32_t>(word);
    std::memcpy(&f, &low, 4);
    return f;
}

}  // namespace

extern "C" int popkv_kv4_write_words(const int64_t* w) {
    return popkv_kv4_write(at<const popkv_kv4_cache>(w[0]), w[1], at<const int32_t>(w[2]), w[3], at<const int32_t>(w[4]),
                           at<const void>(w[5]), at<const void>(w[6]), static_cast<int>(w[7]), w[8], w[9], w[10], w[11],
                           w[12], w[13], w[14], at<void>(w[15]));
}

extern "C" int popkv_kv4_read_words(const int64_t* w) {
    return popkv_kv4_read(at<const popkv_kv4_cache>(w[0]), w[1], at<const int32_t>(w[2]), w[3], w[4], w[5],
                          at<void>(w[6]), at<void>(w[7]), static_cast<int>(w[8]), at<void>(w[9]));
}

extern "C" int popkv_kv4_attention_words(const int64_t* w) {
    return popkv_kv4_attention(at<const popkv_kv4_cache>(w[0]), w[1], at<const int32_t>(w[2]), w[3],
                               at<const int32_t>(w[4]), at<const void>(w[5]), static_cast<int>(w[6]), w[7], w[8], w[9],
                               w[10], w[11], float_of(w[12]), at<void>(w[13]), w[14], at<void>(w[15]), at<void>(w[16]));
}

extern "C" int popkv_kv4_attention_selected_words(const int64_t* w) {
    return popkv_kv4_attention_selected(at<const popkv_kv4_cache>(w[0]), w[1], at<const int32_t>(w[2]), w[3],
                                        at<const void>(w[4]), static_cast<int>(w[5]), w[6], w[7], w[8],
                                        at<const int64_t>(w[9]), w[10], at<const uint8_t>(w[11]), float_of(w[12]),
                                        at<void>(w[13]), w[14], at<void>(w[15]), at<void>(w[16]));
}

extern "C" int popkv_verify_drafts_words(const int64_t* w) {
    return popkv_verify_drafts(at<const void>(w[0]), w[1], w[2], at<const void>(w[3]), w[4], w[5], static_cast<int>(w[6]),
                               w[7], w[8], w[9], at<const int64_t>(w[10]), at<const int32_t>(w[11]),
                               at<const float>(w[12]), at<const float>(w[13]), at<void>(w[14]), at<int64_t>(w[15]),
                               at<int32_t>(w[16]), at<void>(w[17]));
}
