// Execution engine of the emulated model operators (see hip/hip_runtime.h in this directory): test infrastructure only.
#include <hip/hip_runtime.h>
#include <sanitizer/common_interface_defs.h>
#include <stdio.h>
#include <sys/mman.h>

#include <mutex>
#include <random>
#include <vector>

// Saves the registers a callee has to keep on the running stack, leaves the stack's end in *save and goes on from `to`.
extern "C" void LanesSwitch(void** save, void* to);
asm(R"(
.text
.globl LanesSwitch
.hidden LanesSwitch
.type LanesSwitch,@function
LanesSwitch:
    pushq %rbp
    pushq %rbx
    pushq %r12
    pushq %r13
    pushq %r14
    pushq %r15
    movq %rsp, (%rdi)
    movq %rsi, %rsp
    popq %r15
    popq %r14
    popq %r13
    popq %r12
    popq %rbx
    popq %rbp
    retq
.size LanesSwitch,.-LanesSwitch
)");

#if defined(__has_feature)
#if __has_feature(address_sanitizer)
#define LANES_ASAN 1
#endif
#endif

namespace lanes {

Idx g_thread = {0, 0, 0}, g_block = {0, 0, 0};

namespace {

constexpr unsigned kWave = 64;
constexpr size_t kStack = 256 * 1024;
enum State { READY, EXCHANGE, BARRIER, DONE };

struct Lane {
    void* sp;
    uint8_t* stack;
    void* fake;           // the sanitizer's record of the fiber's stack
    State state;
    int site;
    unsigned exchanges;   // so far
};
struct Wave {
    uint32_t value[2][kWave];     // of this exchange and the one before, which slower lanes still read
    uint64_t active[2];
};

std::vector<Lane> g_lanes;
std::vector<Wave> g_waves;
unsigned g_current;
void* g_home;
void* g_homeFake;
const void* g_homeStack;
size_t g_homeSize;
const std::function<void()>* g_body;
std::vector<uint8_t> g_lds;
std::mutex g_mutex;
std::mt19937 g_random(1);

[[noreturn]] void Die(const char* what, int site)
{
    fprintf(stderr, "emulated kernel: %s (workgroup %u, lane %u, line %d)\n", what, g_block.x, g_current, site);
    abort();
}

void ToHome(bool last)
{
    Lane& l = g_lanes[g_current];
    (void)last;
#ifdef LANES_ASAN
    __sanitizer_start_switch_fiber(last ? nullptr : &l.fake, g_homeStack, g_homeSize);
#endif
    LanesSwitch(&l.sp, g_home);
#ifdef LANES_ASAN
    __sanitizer_finish_switch_fiber(l.fake, &g_homeStack, &g_homeSize);
#endif
}

void Entry()
{
#ifdef LANES_ASAN
    __sanitizer_finish_switch_fiber(nullptr, &g_homeStack, &g_homeSize);
#endif
    (*g_body)();
    g_lanes[g_current].state = DONE;
    ToHome(true);
    abort();
}

void Resume(unsigned i)
{
    Lane& l = g_lanes[i];
    g_current = i;
    g_thread.x = i;
#ifdef LANES_ASAN
    __sanitizer_start_switch_fiber(&g_homeFake, l.stack, kStack);
#endif
    LanesSwitch(&g_home, l.sp);
#ifdef LANES_ASAN
    __sanitizer_finish_switch_fiber(g_homeFake, nullptr, nullptr);
#endif
}

// Runs one wavefront until all of its lanes wait at a barrier or have left.
void RunWave(unsigned wave, unsigned lanes)
{
    const unsigned first = wave * kWave, end = first + kWave < lanes ? first + kWave : lanes;
    for (;;) {
        for (unsigned i = first; i < end; ++i) {
            if (g_lanes[i].state == READY) {
                Resume(i);
            }
        }
        uint64_t active = 0;
        unsigned some = end;
        for (unsigned i = first; i < end; ++i) {
            if (g_lanes[i].state == EXCHANGE) {
                active |= 1ull << (i - first);
                some = i;
            }
        }
        if (active == 0) {
            return;
        }
        for (unsigned i = first; i < end; ++i) {
            Lane& l = g_lanes[i];
            if (l.state == EXCHANGE) {
                if (l.site != g_lanes[some].site || l.exchanges != g_lanes[some].exchanges) {
                    g_current = i;
                    Die("lanes of a wavefront at different cross-lane operations", l.site);
                }
                l.state = READY;
            }
        }
        g_waves[wave].active[g_lanes[some].exchanges & 1] = active;
    }
}

void RunGroup(unsigned lanes)
{
    const unsigned waves = (lanes + kWave - 1) / kWave;
    for (unsigned i = 0; i < lanes; ++i) {
        Lane& l = g_lanes[i];
        void** top = reinterpret_cast<void**>(l.stack + kStack);
        top -= 2;
        *top = reinterpret_cast<void*>(&Entry);       // return address; the entry then has the alignment of a call
        top -= 6;
        l.sp = top;
        l.state = READY;
        l.exchanges = 0;
        l.fake = nullptr;
    }
    for (;;) {
        std::vector<unsigned> order(waves);
        for (unsigned w = 0; w < waves; ++w) {
            order[w] = w;
        }
        for (unsigned w = waves; w > 1; --w) {
            std::swap(order[w - 1], order[g_random() % w]);
        }
        for (unsigned w : order) {
            RunWave(w, lanes);
        }
        bool waiting = false;
        for (unsigned i = 0; i < lanes; ++i) {
            if (g_lanes[i].state == BARRIER) {
                g_lanes[i].state = READY;
                waiting = true;
            }
        }
        if (!waiting) {
            return;
        }
    }
}

}  // namespace

void Launch(dim3 grid, dim3 block, size_t ldsBytes, const std::function<void()>& body)
{
    std::lock_guard<std::mutex> guard(g_mutex);
    if (grid.y != 1 || grid.z != 1 || block.y != 1 || block.z != 1 || block.x == 0 || block.x > 1024 || grid.x == 0 ||
        static_cast<uint64_t>(grid.x) * block.x >= 1ull << 32) {
        Die("launch dimensions", 0);
    }
    while (g_lanes.size() < block.x) {
        Lane l = {};
        l.stack = static_cast<uint8_t*>(mmap(nullptr, kStack, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
        g_lanes.push_back(l);
    }
    g_waves.assign((block.x + kWave - 1) / kWave, Wave{});
    g_body = &body;
    for (unsigned b = 0; b < grid.x; ++b) {
        g_block.x = b;
        std::vector<uint8_t>(ldsBytes, static_cast<uint8_t>(0xA5 + b)).swap(g_lds);      // LDS holds anything at the start
        RunGroup(block.x);
    }
}

void* DynamicLds() { return g_lds.data(); }

void SyncThreads()
{
    g_lanes[g_current].state = BARRIER;
    ToHome(false);
}

const uint32_t* Exchange(uint32_t value, int site, uint64_t* active, unsigned* lane)
{
    Lane& l = g_lanes[g_current];
    Wave& w = g_waves[g_current / kWave];
    const unsigned turn = ++l.exchanges & 1;
    *lane = g_current % kWave;
    w.value[turn][*lane] = value;
    l.state = EXCHANGE;
    l.site = site;
    ToHome(false);
    *active = w.active[turn];
    return w.value[turn];
}

uint32_t UpdateDpp(uint32_t old, uint32_t src, int control, int rowMask, int bankMask, bool boundControl, int site)
{
    uint64_t active;
    unsigned lane;
    const uint32_t* v = Exchange(src, site, &active, &lane);
    const unsigned row = lane / 16, in = lane % 16;
    if (((rowMask >> row) & 1) == 0 || ((bankMask >> (in / 4)) & 1) == 0) {
        return old;
    }
    int from = -1;
    if (control >= 0 && control <= 0xFF) {                  // permutation within four lanes
        from = static_cast<int>((lane & ~3u) | ((static_cast<unsigned>(control) >> (2 * (lane & 3))) & 3u));
    } else if (control >= 0x111 && control <= 0x11F) {      // from lower lanes of the row
        const int n = control & 15;
        from = static_cast<int>(in) >= n ? static_cast<int>(lane) - n : -1;
    } else if (control >= 0x121 && control <= 0x12F) {      // rotated within the row
        from = static_cast<int>(row * 16 + ((in + 16 - (control & 15)) & 15));
    } else if (control == 0x140) {
        from = static_cast<int>(row * 16 + 15 - in);
    } else if (control == 0x141) {
        from = static_cast<int>((lane & ~7u) + 7 - (lane & 7));
    } else if (control == 0x142) {                          // the last lane of the row before
        from = row == 0 ? -1 : static_cast<int>(row * 16 - 1);
    } else if (control == 0x143) {                          // lane 31
        from = row < 2 ? -1 : 31;
    } else {
        Die("control of a lane permutation", site);
    }
    if (from < 0) {
        return boundControl ? 0 : old;
    }
    if (((active >> from) & 1) == 0) {
        Die("a lane that takes no part is read", site);
    }
    return v[from];
}

uint64_t Ballot(bool value, int site)
{
    uint64_t active, all = 0;
    unsigned lane;
    const uint32_t* v = Exchange(value ? 1 : 0, site, &active, &lane);
    for (unsigned i = 0; i < kWave; ++i) {
        all |= static_cast<uint64_t>(((active >> i) & 1) && v[i]) << i;
    }
    return all;
}

uint32_t ReadLane(uint32_t v, uint32_t from, int site)
{
    uint64_t active;
    unsigned lane;
    const uint32_t* all = Exchange(v, site, &active, &lane);
    if (from >= kWave || ((active >> from) & 1) == 0) {
        Die("a lane that takes no part is read", site);
    }
    return all[from];
}

uint32_t ReadFirstLane(uint32_t v, int site)
{
    uint64_t active;
    unsigned lane;
    const uint32_t* all = Exchange(v, site, &active, &lane);
    return all[__builtin_ctzll(active)];
}

uint32_t ShuffleXor(uint32_t v, unsigned distance, int site)
{
    uint64_t active;
    unsigned lane;
    const uint32_t* all = Exchange(v, site, &active, &lane);
    if (((active >> (lane ^ distance)) & 1) == 0) {
        Die("a lane that takes no part is read", site);
    }
    return all[lane ^ distance];
}

// The rows of `distance` lanes that are odd in `a` change places with those that are even in `b`.
Pair SwapRows(uint32_t a, uint32_t b, unsigned distance, int site)
{
    uint64_t active;
    unsigned lane;
    const uint32_t* v = Exchange(a, site, &active, &lane);
    const uint32_t* w = Exchange(b, site, &active, &lane);
    const unsigned other = lane ^ distance;
    if (((active >> other) & 1) == 0) {
        Die("a lane that takes no part is read", site);
    }
    const bool odd = (lane & distance) != 0;
    return Pair{odd ? w[other] : a, odd ? b : v[other]};
}

float WidenFp8(int word, int byte)
{
    const unsigned code = (static_cast<unsigned>(word) >> (8 * byte)) & 0xFFu;
    const int exponent = static_cast<int>((code >> 3) & 15u), digits = static_cast<int>(code & 7u);
    float v = exponent == 0 ? ldexpf(static_cast<float>(digits), -9) : ldexpf(static_cast<float>(8 + digits), exponent - 10);
    if ((code & 0x7Fu) == 0x7Fu) {
        v = __builtin_nanf("");
    }
    return (code & 0x80u) != 0 ? -v : v;
}

namespace {
unsigned NarrowFp8(float x)
{
    const float v = fabsf(x);
    if (x != x) {
        return 0x7Fu;
    }
    if (v >= 464.0f) {      // would round to 480
        Die("a value beyond the FP8 type's range", 0);
    }
    unsigned best = 0;
    for (unsigned code = 1; code < 0x7Fu; ++code) {
        const float to = fabsf(WidenFp8(static_cast<int>(code), 0) - v), so = fabsf(WidenFp8(static_cast<int>(best), 0) - v);
        if (to < so || (to == so && (code & 1) == 0)) {
            best = code;
        }
    }
    return best | (signbit(x) ? 0x80u : 0u);
}
}  // namespace

int NarrowFp8Pair(float a, float b, int old, bool upper)
{
    const unsigned pair = NarrowFp8(a) | (NarrowFp8(b) << 8), word = static_cast<unsigned>(old);
    return static_cast<int>(upper ? (word & 0xFFFFu) | (pair << 16) : (word & 0xFFFF0000u) | pair);
}

}  // namespace lanes
