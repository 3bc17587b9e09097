"""The host's page bookkeeping of the batch decoder (csrc/page_book.hpp), built by itself with the host compiler,
against a plain model: random steps, forks and drops, every number compared after each."""
import os
import random
import subprocess

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust-deeplearning_amd", "csrc")
DRIVER = r"""
#include <iostream>
#include "page_book.hpp"
using namespace std;
static vector<int> ints() { size_t n; cin >> n; vector<int> v(n); for (int& x : v) cin >> x; return v; }
int main() {
    rdl::PageBook b;
    string op;
    while (cin >> op) {
        if (op == "begin") { size_t s, p; int page; cin >> s >> p >> page; b.begin(s, p, page); }
        if (op == "step") { auto c = ints(); cout << b.step_pages(c.data()) << ' '; b.step(c.data()); }
        if (op == "fork") { auto p = ints(), c = ints(); cout << b.fork_pages(p.data(), p.size()) << ' '; b.fork(p.data(), c.data(), p.size()); }
        if (op == "drop") { size_t s; cin >> s; b.drop(s); }
        for (int x : b.len) cout << x << ' ';
        cout << "| ";
        for (int x : b.free) cout << x << ' ';
        cout << "| ";
        for (int x : b.holders) cout << x << ' ';
        for (size_t s = 0; s < b.len.size(); s++) {
            cout << "| ";
            for (size_t p = 0; p < b.pages_of(b.len[s]); p++) cout << b.row(s)[p] << ' ';
        }
        cout << endl;
    }
}
"""


class Plain:
    """Rows as lists; a page is free when no row names it."""

    def __init__(self, n_seq, pages, page):
        self.page, self.rows, self.len, self.free = page, [[] for _ in range(n_seq)], [0] * n_seq, list(range(pages))
        self.pages = pages

    def wanted(self, counts):
        return sum(-(-(n + c) // self.page) - len(r) for n, c, r in zip(self.len, counts, self.rows))

    def step(self, counts):
        k = self.wanted(counts)
        for b, c in enumerate(counts):
            self.len[b] += c
            while len(self.rows[b]) * self.page < self.len[b]:
                self.rows[b].append(self.free.pop(0))
        return k

    def fork(self, parents, children):
        k = 0
        for p, c in zip(parents, children):
            self.rows[c], self.len[c] = list(self.rows[p]), self.len[p]
            if self.len[p] % self.page:
                self.rows[c][-1] = self.free.pop(0)
                k += 1
        return k

    def drop(self, s):
        held, self.rows[s], self.len[s] = self.rows[s], [], 0
        self.free += [p for p in held if all(p not in r for r in self.rows)]

    def state(self):
        holders = [sum(p in r for r in self.rows) for p in range(self.pages)]
        assert sorted(self.free) == [p for p in range(self.pages) if not holders[p]]
        return " | ".join(" ".join(map(str, x)) for x in (self.len, self.free, holders, *self.rows))


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    d = tmp_path_factory.mktemp("book")
    (d / "driver.cpp").write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-D_GLIBCXX_ASSERTIONS", "-I", SRC, str(d / "driver.cpp"),
                    "-o", str(d / "driver")], check=True)
    return str(d / "driver")


@pytest.mark.parametrize("seed,n_seq,pages,page", [(1, 1, 3, 64), (2, 6, 24, 16), (3, 40, 90, 16), (4, 9, 9, 64), (5, 17, 400, 16)])
def test_random_steps_forks_and_drops(driver, seed, n_seq, pages, page):
    r = random.Random(seed)
    m = Plain(n_seq, pages, page)
    says, want = [f"begin {n_seq} {pages} {page}"], [m.state()]
    for _ in range(300):
        what = r.random()
        took = ""
        if what < 0.5:
            counts = [r.choice([0, 1, page - 1, page, r.randrange(3 * page)]) if r.random() < 0.4 else 0 for _ in range(n_seq)]
            if m.wanted(counts) > len(m.free) or any(n + c > pages * page for n, c in zip(m.len, counts)):
                continue
            says.append(f"step {n_seq} " + " ".join(map(str, counts)))
            took = str(m.step(counts))
        elif what < 0.75:
            empty = [s for s in range(n_seq) if m.len[s] == 0]
            full = [s for s in range(n_seq) if m.len[s]]
            if not empty or not full:
                continue
            children = r.sample(empty, r.randint(1, len(empty)))
            parents = [r.choice(full) for _ in children]
            if sum(m.len[p] % page != 0 for p in parents) > len(m.free):
                continue
            says.append(f"fork {len(parents)} {' '.join(map(str, parents))} {len(children)} {' '.join(map(str, children))}")
            took = str(m.fork(parents, children))
        else:
            s = r.randrange(n_seq)
            says.append(f"drop {s}")
            m.drop(s)
        want.append((took + " " + m.state()).strip())
    assert len(want) > 60 or n_seq == 1
    got = subprocess.run([driver], input="\n".join(says), text=True, capture_output=True, check=True).stdout.splitlines()
    assert [" ".join(g.split()) for g in got] == [" ".join(w.split()) for w in want]
