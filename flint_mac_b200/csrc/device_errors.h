// What flint_attn_check makes of the error words that kernels leave on the device.  Host code without CUDA, so that a test can
// put a fake in the place of the device's words.
#pragma once

#include <string>

namespace flint {

// Reads and clears every word before anything is said about the first one, so that an error is reported once and nothing of it
// is left for the launches after it: a decode launch that gave up leaves its arrival counters partly counted, and a later
// launch would merge too early.  Returns the messages of all words that were set, or an empty string.
//   int take_prefill(), take_decode(), take_exchange()  read a word and clear it (0: nothing happened)
//   void clear_counters()                               the decode kernels' arrival counters back to zero
template <typename Words>
std::string take_device_errors(Words &&words) {
    const int prefill = words.take_prefill(), decode = words.take_decode(), exchange = words.take_exchange();
    if (decode) words.clear_counters();
    std::string all;
    auto add = [&](const std::string &what) { all += (all.empty() ? "" : "; ") + what; };
    if (prefill) add("prefill kernel reported device error " + std::to_string(prefill));
    if (decode) add("decode kernel reported device error " + std::to_string(decode));
    if (exchange) add("the wait for a peer's partial records ran out (exchange error " + std::to_string(exchange) + ")");
    return all;
}

}  // namespace flint
