"""The host arithmetic that tells whether a call's tensors share elements (csrc/g4q_overlap.h), compiled with the host
compiler, against sets of elements."""
import itertools
import random
import subprocess

import pytest

from conftest import ROOT

D = 8

PROGRAM = r"""
#include <cstdio>
#include <string>
#include "g4q_overlap.h"
int main(int argc, char** argv) {
    G4qPagedCache c;
    long long k, v, n, ps, hs, ss, at, m, ts, rs;
    G4qHeadRows r, o;
    const std::string mode = argc > 1 ? argv[1] : "";
    while (mode == "apart" && std::scanf("%lld %d %lld %lld", &m, &r.n_heads, &ts, &rs) == 4) {
        r.token_stride = ts, r.head_stride = rs;
        std::printf("%d\n", (int)g4q::rows_apart(r, m, 8));
    }
    while (mode == "pair" && std::scanf("%lld %lld %d %lld %lld %lld %d %lld %lld", &m, &k, &r.n_heads, &ts, &rs, &v, &o.n_heads,
                                        &ps, &hs) == 9) {
        r.data = (uint16_t*)0 + k, r.token_stride = ts, r.head_stride = rs;
        o.data = (uint16_t*)0 + v, o.token_stride = ps, o.head_stride = hs;
        std::printf("%d\n", (int)g4q::rows_meet(r, o, m, 8));
    }
    while (mode != "pair" && mode != "apart" && std::scanf("%lld %lld %lld %d %d %lld %lld %lld", &k, &v, &n, &c.page_size, &c.n_kv_heads, &ps, &hs, &ss) == 8) {
        c.k = (uint16_t*)0 + k, c.v = (uint16_t*)0 + v;
        c.n_pages = n, c.head_dim = 8;
        c.page_stride = ps, c.head_stride = hs, c.slot_stride = ss;
        const char* wrong = g4q::shared_slots(c);
        if (mode == "rows") {      // and rows: meets the cache or not
            if (std::scanf("%lld %lld %d %lld %lld", &at, &m, &r.n_heads, &ts, &rs) != 5) return 1;
            r.data = (uint16_t*)0 + at, r.token_stride = ts, r.head_stride = rs;
            wrong = g4q::meets_cache(r, m, c, g4q::cache_lattice(c)) ? "meets" : nullptr;
        }
        std::printf("%d %s\n", (int)g4q::cache_lattice(c).nested(), wrong ? wrong : "-");
    }
}
"""


@pytest.fixture(scope="module")
def answers(tmp_path_factory):
    """Runs the program on cases, numbers each: (k, v, pages, page_size, heads, page_stride, head_stride, slot_stride) gives
    (nested, what is wrong). Mode "rows": the cases go on with (data, tokens, heads, token_stride, head_stride), and give
    (nested, "meets" or "-"). Mode "apart": (tokens, heads, token_stride, head_stride) gives (apart, "").
    Mode "pair": (tokens, data, heads, token_stride, head_stride, data, heads, token_stride, head_stride) gives (meet, "")."""
    at = tmp_path_factory.mktemp("overlap")
    (at / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    str(ROOT / "include"), "-I", str(ROOT / "helios_b200" / "csrc"), str(at / "main.cpp"), "-o", str(at / "main")],
                   check=True)

    def ask(cases, mode=""):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        out = subprocess.run([str(at / "main"), mode], input=text, check=True, capture_output=True, text=True).stdout.splitlines()
        assert len(out) == len(cases)
        return [(line[0] == "1", line[2:]) for line in out]

    return ask


def rows(base, counts, strides):
    return [base + sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*(range(n) for n in counts))]


def elements(starts):
    return [e for r in starts for e in range(r, r + D)]


def test_caches_against_sets_of_elements(answers):
    """Layouts of all orders with gaps, single axes and shared elements: the refusals are those of the sets, except that
    axes which interleave without sharing are refused too."""
    rng = random.Random(1)
    cases = []
    for _ in range(6000):
        counts = [rng.choice([1, 2, 3]) for _ in range(3)]
        strides = [0, 0, 0]
        inner = D
        for axis in rng.sample(range(3), 3):
            strides[axis] = inner + rng.choice([0, 0, 8, 24]) if rng.random() < 0.9 else 8 * rng.randrange(1, 9)
            inner = max(inner, strides[axis] * counts[axis])
        k = 4096
        cases.append((k, k + 8 * rng.randrange(-24, 25), counts[0], counts[2], counts[1], strides[0], strides[1], strides[2]))
    wrong = {"nested": 0, "shared": 0}
    for (k, v, pages, slots, heads, ps, hs, ss), (nested, text) in zip(cases, answers(cases)):
        ke, ve = (elements(rows(b, (pages, heads, slots), (ps, hs, ss))) for b in (k, v))
        if nested:
            assert len(set(ke)) == len(ke)
            assert (text != "-") == bool(set(ke) & set(ve)), (k, v, pages, slots, heads, ps, hs, ss)
            wrong["shared"] += text == "cache: k and v share elements"
        else:
            assert text == "cache: pages, heads and slots must not overlap"
            wrong["nested"] += 1
        if len(set(ke)) < len(ke) or set(ke) & set(ve):
            assert text != "-"
    assert min(wrong.values()) > 200 and sum(wrong.values()) < 5000


def test_usual_caches_qualify(answers):
    page, heads, pages, d = 16, 2, 4, D
    block = page * heads * d
    usual = [(0, pages * block, pages, page, heads, block, page * d, d),                       # two tensors behind each other
             (0, pages * block, pages, page, heads, block, d, heads * d),                      # slots before heads
             (0, block, pages, page, heads, 2 * block, page * d, d),                           # k and v of a page in turn
             (0, d, pages, page, heads, 2 * block, 2 * page * d, 2 * d),                       # k and v of a slot in turn
             (3 * block, 3 * pages * block + 3 * block, pages, page, heads, 3 * block, page * d, d),   # one layer of three
             (0, 2 ** 40, 2 ** 31 - 2, 65536, 65535, 2 ** 38 - 8, d * 65536, d)]               # far beyond any memory
    got = answers(usual)
    assert [text for _, text in got[:5]] == ["-"] * 5
    assert got[5][1] != "-"


def test_one_tensor_for_keys_and_values(answers):
    """The key projection is the value too in some layers, but what is stored of it is not."""
    assert answers([(64, 64, 3, 16, 1, 128, 128, 8), (64, 64 + 8, 3, 16, 1, 128, 128, 8)]) == \
        [(True, "cache: k and v share elements")] * 2


def test_rows_against_sets_of_elements(answers):
    """Rows before, in, between and behind the slots of a cache. Exact where the cache's axes are nested; else nothing that
    is shared is missed."""
    rng = random.Random(2)
    cases = []
    for _ in range(6000):
        counts = [rng.choice([1, 2, 3]) for _ in range(3)]
        strides = [0, 0, 0]
        inner = D
        for axis in rng.sample(range(3), 3):
            strides[axis] = inner + rng.choice([0, 8, 24, 64]) if rng.random() < 0.95 else 8 * rng.randrange(1, 9)
            inner = max(inner, strides[axis] * counts[axis])
        k, m, heads = 4096, rng.choice([1, 2, 4]), rng.choice([1, 2])
        cases.append((k, k + 8 * rng.randrange(-24, 25), counts[0], counts[2], counts[1], strides[0], strides[1], strides[2],
                      k + 8 * rng.randrange(-40, 80), m, heads, 8 * rng.randrange(0, 9), 8 * rng.randrange(1, 9)))
    seen = {False: 0, True: 0}
    for case, (nested, text) in zip(cases, answers(cases, "rows")):
        k, v, pages, slots, heads, ps, hs, ss, at, m, row_heads, ts, rs = case
        held = set(elements(rows(k, (pages, heads, slots), (ps, hs, ss)) + rows(v, (pages, heads, slots), (ps, hs, ss))))
        meets = bool(held & set(elements(rows(at, (m, row_heads), (ts, rs)))))
        assert text == ("meets" if meets else "-") if nested else meets <= (text == "meets"), case
        seen[meets] += nested
    assert min(seen.values()) > 1000


def test_rows_of_an_output_against_sets_of_elements(answers):
    rng = random.Random(3)
    cases = [(rng.randrange(1, 6), rng.randrange(1, 6), 8 * rng.randrange(0, 9), 8 * rng.randrange(0, 9)) for _ in range(5000)]
    for (m, heads, ts, hs), (apart, _) in zip(cases, answers(cases, "apart")):
        held = elements(rows(0, (m, heads), (ts, hs)))
        assert apart == (len(set(held)) == len(held)), (m, heads, ts, hs)
    many = 2 ** 20          # the fourth: heads 24 = 16 + 8 on lie in the gaps between the tokens' rows
    assert [a for a, _ in answers([(many, 16, 128, 8), (many, 16, 8, 8 * many), (many, 16, 8, 8), (many, 2, 16, 8 * 3),
                                   (many, 1, 0, 0), (1, 16, 0, 8), (many, many, 2 ** 40, 2 ** 41)], "apart")] == \
        [True, True, False, True, False, True, False]


def test_two_tensors_of_rows_against_sets_of_elements(answers):
    """Exact where one of the two has no rows that overlap; else nothing that is shared is missed."""
    rng = random.Random(4)
    cases = []
    for _ in range(20000):
        m, at = rng.randrange(1, 5), 4096
        strides = []
        for _ in range(2):
            heads, inner = rng.randrange(1, 5), 8 * rng.choice([1, 1, 2, 3])
            tokens_out = rng.random() < 0.6
            outer = inner * (heads if tokens_out else m) + 8 * rng.randrange(-1, 7)
            strides.append((heads, outer, inner) if tokens_out else (heads, inner, outer))
        if rng.random() < 0.5:
            strides[1] = (strides[1][0], *strides[0][1:])
        cases.append((m, at, *strides[0], at + 8 * rng.randrange(-30, 31), *strides[1]))
    seen = [0, 0, 0]
    for case, (meet, _) in zip(cases, answers(cases, "pair")):
        m, a, na, ta, ha, b, nb, tb, hb = case
        ea, eb = elements(rows(a, (m, na), (ta, ha))), elements(rows(b, (m, nb), (tb, hb)))
        real = bool(set(ea) & set(eb))
        assert meet or not real, case
        if len(set(ea)) < len(ea) and len(set(eb)) < len(eb):
            continue
        interleaved = min(len(set(ea)), len(set(eb))) and (max(ea) > min(eb) and max(eb) > min(ea)) and not real
        seen[0 if real else 2 if interleaved else 1] += 1
        nested = [t >= h * (n - 1) + D or h >= t * (m - 1) + D or n == 1 or m == 1 for n, t, h in ((na, ta, ha), (nb, tb, hb))]
        assert meet == real or not any(nested), case
    assert min(seen) > 1000, seen
