// paged.cpp - the entry points over paged caches on the host (device.hpp).  Reads calls from the standard input, a line
// each; buffers are allocations of their own of exactly the given size:
//   buf NAME BYTES FILE      (FILE -: every byte 0xA5)
//   save NAME FILE
//   order 1|-1               blocks and waves in the order of their number, or backwards and in turn
//   pages TYPE NKV HD PAGE PAGES OPENS k v k_scale v_scale k_open v_open
//   step SEQS ROWS MAX_ROWS MAX_PAGES row0 past table open
//   rotary cs POSITIONS ROTARY_DIM AXES INTERLEAVED pos SECTION ..
//   prep GATED NQ EPS SRC_STRIDE OUT_STRIDE src q_norm k_norm q gate     (k and v behind q in a row of src)
//   read OUT_TYPE k v
//   attention NQ Q_STRIDE OUT_STRIDE q gate out
//   logprobs TYPE LD ROWS VOCAB INV_TEMPERATURE TOP logits tokens logprob entropy rank top top_logprob
//   codes FILE               of fp16 values up to fp16 maxima: how many have a code that is not the nearest
// Names of nothing are 0.
#include "device.hpp"

#include <fstream>
#include <iostream>
#include <map>
#include <sstream>
#include <string>
#include <vector>

#include "xqhip.h"
#include "xqhip_kernels.hpp"

#include "paged_cache.hip"

#include "paged_attn.hip"

#include "paged_api.hip"

namespace xqhip {
void set_last_error(const std::string& msg) { std::cerr << msg << "\n"; }
}  // namespace xqhip

namespace {

struct Buffer {
    char* at;
    size_t bytes;
};
std::map<std::string, Buffer> buffers;

void* at(const std::string& name) {
    if (name == "0") return nullptr;
    if (!buffers.count(name)) {
        std::cerr << "no buffer " << name << "\n";
        std::exit(2);
    }
    return buffers[name].at;
}
template <typename T>
T* as(const std::string& name) {
    return static_cast<T*>(at(name));
}
Buffer allocate(size_t n) {
    Buffer b{static_cast<char*>(std::malloc(n ? n : 1)), n};  // (16-byte aligned, an end of its own)
    std::memset(b.at, 0xA5, n);
    return b;
}

// Codes of 8-bit pages against the quotient in 64 bits: ties are exact in both.
int64_t wrong_codes() {
    int64_t wrong = 0;
    for (uint32_t m = 1; m < 0x7c00; ++m) {
        // significands of normal maxima repeat with every exponent: all of one, every 61st of the others
        if ((m < 0x3c00 || m >= 0x4000) && m >= 0x400 && m % 61) continue;
        const float mx = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(m))), inv = 1.0f / mx;
        for (uint32_t v = 0; v <= m; ++v) {
            const _Float16 x = __builtin_bit_cast(_Float16, static_cast<uint16_t>(v));
            const double want = rint(127.0 * static_cast<double>(x) / static_cast<double>(mx));
            wrong += xqhip::code_of(x, mx, inv) != static_cast<int>(want) || xqhip::code_of(-x, mx, inv) != -static_cast<int>(want);
        }
    }
    return wrong;
}

}  // namespace

int main() {
    std::string line;
    xqhip_pages kv{};
    xqhip_step step{};
    xqhip_rotary rot{};
    bool turned = false;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        std::string what, name, file;
        in >> what;
        auto next = [&] {
            std::string s;
            in >> s;
            return s;
        };
        auto number = [&] { return std::stoi(next()); };
        int rc = 0;
        if (what == "buf") {
            size_t n;
            in >> name >> n >> file;
            buffers[name] = allocate(n);
            if (file != "-") {
                std::ifstream f(file, std::ios::binary);
                f.read(buffers[name].at, static_cast<std::streamsize>(n));
                if (static_cast<size_t>(f.gcount()) != n) return 2;
            }
        } else if (what == "save") {
            in >> name >> file;
            std::ofstream(file, std::ios::binary).write(as<char>(name), static_cast<std::streamsize>(buffers[name].bytes));
        } else if (what == "order") {
            host::order = number();
        } else if (what == "pages") {
            kv.type = number();
            kv.nkv = number();
            kv.head_dim = number();
            kv.page = number();
            kv.pages = number();
            kv.opens = number();
            kv.k = at(next());
            kv.v = at(next());
            kv.k_scale = as<float>(next());
            kv.v_scale = as<float>(next());
            kv.k_open = at(next());
            kv.v_open = at(next());
        } else if (what == "step") {
            step.seqs = number();
            step.rows = number();
            step.max_rows = number();
            step.max_pages = number();
            step.row0 = as<int32_t>(next());
            step.past = as<int32_t>(next());
            step.table = as<int32_t>(next());
            step.open = as<int32_t>(next());
        } else if (what == "rotary") {
            const float* cs = as<float>(next());
            const int positions = number(), dim = number(), axes = number(), interleaved = number();
            const int32_t* pos = as<int32_t>(next());
            int32_t sections[4] = {};
            for (int a = 0; a < axes; ++a) sections[a] = number();
            rc = xqhip_rotary_init(cs, positions, dim, sections, axes, interleaved, pos, &rot);
            turned = true;
        } else if (what == "prep") {
            const int gated = number(), nq = number();
            const float eps = std::strtof(next().c_str(), nullptr);
            const int src_stride = number(), out_stride = number(), q_width = nq * kv.head_dim * (gated ? 2 : 1);
            const float* src = as<float>(next());
            const float* qn = as<float>(next());
            const float* kn = as<float>(next());
            float* q = as<float>(next());
            float* gate = as<float>(next());
            rc = xqhip_attn_prep_paged(src, src + q_width, src + q_width + kv.nkv * kv.head_dim, gated, nq, qn, kn, eps, turned ? &rot : nullptr,
                                       &step, src_stride, out_stride, q, gate, &kv, nullptr);
        } else if (what == "read") {
            const int type = number();
            void* k = at(next());
            void* v = at(next());
            rc = xqhip_paged_read(&kv, &step, type, k, v, nullptr);
        } else if (what == "attention") {
            const int nq = number(), q_stride = number(), out_stride = number();
            const float* q = as<float>(next());
            const float* gate = as<float>(next());
            float* out = as<float>(next());
            Buffer ws = allocate(xqhip_paged_attention_workspace_bytes(nq, kv.nkv, kv.head_dim));
            rc = xqhip_paged_attention(q, gate, &kv, nq, &step, q_stride, out, out_stride, ws.at, ws.bytes, nullptr);
            std::free(ws.at);
        } else if (what == "logprobs") {
            const int type = number(), ld = number(), rows = number(), vocab = number();
            const float inv_t = std::strtof(next().c_str(), nullptr);
            const int top = number();
            const void* x = at(next());
            const int32_t* tokens = as<int32_t>(next());
            float* logprob = as<float>(next());
            float* entropy = as<float>(next());
            int32_t* rank = as<int32_t>(next());
            int32_t* ids = as<int32_t>(next());
            float* top_logprob = as<float>(next());
            Buffer ws = allocate(xqhip_token_logprobs_workspace_bytes(rows, vocab, top));
            rc = xqhip_token_logprobs(x, type, ld, rows, vocab, inv_t, tokens, top, logprob, entropy, rank, ids, top_logprob, ws.at, ws.bytes, nullptr);
            std::free(ws.at);
        } else if (what == "codes") {
            std::ofstream(next()) << wrong_codes();
        } else {
            return 2;
        }
        if (rc != 0) {
            std::cerr << "refused: " << line << "\n";
            return 3;
        }
    }
    return 0;
}
