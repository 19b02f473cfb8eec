"""How `paged_attention` joins the parts of rows that several lots hold (csrc/join_plan.h), compiled for the
host: every slot of a lot has one writer, every part is joined once, and every field of a lock word counts
arrivals of one kind."""

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "chord_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <map>
#include <random>
#include <set>
#include <string>
#include <utility>
#include <vector>
#include "join_plan.h"
using namespace chord;

struct Span { int first, lots; };  // a row's lots

// Rows of `steps` steps, numbered through and cut into lots of `piece` steps.
static std::vector<Span> numbered(const std::vector<long long>& steps, long long piece) {
  std::vector<Span> rows;
  long long at = 0;
  for (long long n : steps) {
    if (n == 0) continue;
    rows.push_back({int(at / piece), int((at + n - 1) / piece - at / piece + 1)});
    at += n;
  }
  return rows;
}

// Rows cut into lots of their own.
static std::vector<Span> apart(const std::vector<long long>& steps, long long piece) {
  std::vector<Span> rows;
  int lot = 0;
  for (long long n : steps) {
    if (n == 0) continue;
    rows.push_back({lot, int((n + piece - 1) / piece)});
    lot += rows.back().lots;
  }
  return rows;
}

static const char* check(const std::vector<Span>& rows) {
  std::map<std::pair<int, int>, std::string> holds;          // (lot, slot): what was written there
  std::map<std::pair<int, int>, std::pair<int, int>> words;  // (lot, field): (row, arrivals expected)
  for (size_t r = 0; r < rows.size(); ++r) {
    const RowJoin join(rows[r].first, rows[r].lots);
    if (rows[r].lots < 2) continue;
    if (join.groups() > kFan || (join.fan > 1 && join.groups() < 2)) return "a last join of too many or of one";
    auto name = [&](int from, int to) { return std::to_string(r) + ":" + std::to_string(from) + "-" + std::to_string(to); };
    auto write = [&](int lot, int slot, const std::string& what) { return slot >= 0 && slot < kSlots && holds.emplace(std::make_pair(lot, slot), what).second; };
    for (int i = 0; i < rows[r].lots; ++i) {
      if (!write(rows[r].first + i, i == 0 ? kSlotFirst : kSlotInside, name(i, i + 1))) return "two parts in one slot";
    }
    if (!words.emplace(std::make_pair(rows[r].first, 1), std::make_pair(int(r), join.groups())).second) return "two rows count in one field";
    std::set<int> begun;
    for (int i = 0; i < rows[r].lots; ++i) {
      const int begin = join.group_of(rows[r].first + i), count = join.group_lots(begin);
      if (i < begin || i >= begin + count || count > kFan) return "not in its group";
      if (count == 1 || !begun.insert(begin).second) continue;
      if (!words.emplace(std::make_pair(rows[r].first + begin, 0), std::make_pair(int(r), count)).second) return "two groups count in one field";
      for (int j = 0; j < count; ++j) {
        const PartPlace at = join.part(begin, j);
        const auto found = holds.find({at.lot, at.slot});
        if (found == holds.end() || found->second != name(begin + j, begin + j + 1)) return "a group joins what is not its part";
      }
      if (!write(rows[r].first + begin, kSlotGroup, name(begin, begin + count))) return "two joins in one slot";
    }
  }
  for (size_t r = 0; r < rows.size(); ++r) {  // after all have written
    const RowJoin join(rows[r].first, rows[r].lots);
    if (rows[r].lots < 2) continue;
    int next = 0;
    for (int j = 0; j < join.groups(); ++j) {
      const PartPlace at = join.joined(j);
      const auto found = holds.find({at.lot, at.slot});
      if (found == holds.end()) return "a last join of nothing";
      const int count = join.group_lots(next);
      if (found->second != std::to_string(r) + ":" + std::to_string(next) + "-" + std::to_string(next + count)) return "a last join of another row's part, or out of order";
      next += count;
    }
    if (next != rows[r].lots) return "parts left out";
  }
  return nullptr;
}

int main() {
  std::mt19937_64 rng(7);
  auto draw = [&](long long low, long long high) { return std::uniform_int_distribution<long long>(low, high)(rng); };
  for (int lots = 1; lots <= 480; ++lots) {
    for (int first : {0, 1, 7, 33}) {
      if (const char* wrong = check({{first, lots}})) return std::printf("%s: %d lots from %d\n", wrong, lots, first), 1;
    }
    // neighbours that share a lot, of every two sizes
    for (int more = 1; more <= 480 - lots + 1; more += 1 + more / 16) {
      if (const char* wrong = check({{0, lots}, {lots - 1, more}})) return std::printf("%s: %d and %d lots\n", wrong, lots, more), 1;
    }
  }
  long long shared = 0;
  for (int trial = 0; trial < 6000; ++trial) {
    const int heads = int(draw(1, 16)), ctas = int(draw(1, 4)) * 120, step = draw(0, 1) ? 16 : 32;
    const int longs = int(draw(0, 3)), shorts = int(draw(0, 64));
    std::vector<long long> steps;
    for (int b = 0; b < longs + shorts; ++b) {
      const long long tokens = b < longs ? draw(1000, 150000) : draw(0, 600);
      steps.push_back((tokens + step - 1) / step);
    }
    std::shuffle(steps.begin(), steps.end(), rng);
    std::vector<long long> rows;
    for (long long n : steps) rows.insert(rows.end(), heads, n);
    long long total = 0;
    for (long long n : rows) total += n;
    if (total == 0) continue;
    const long long piece = 4 * ((total + 4 * ctas - 1) / (4 * ctas));
    const auto spans = numbered(rows, piece);
    for (size_t r = 0; r + 1 < spans.size(); ++r) shared += spans[r].lots > kAtOnce && spans[r + 1].lots > kAtOnce && spans[r].first + spans[r].lots - 1 == spans[r + 1].first;
    if (const char* wrong = check(spans)) return std::printf("%s: trial %d\n", wrong, trial), 1;
    long long own = piece;
    while (true) {
      const auto each = apart(rows, own);
      if (each.back().first + each.back().lots <= ctas) {
        if (const char* wrong = check(each)) return std::printf("%s: trial %d, lots of their own\n", wrong, trial), 1;
        break;
      }
      if (rows.size() > size_t(ctas)) break;
      own *= 2;
    }
  }
  if (shared < 500) return std::printf("only %lld pairs of long rows that share a lot\n", shared), 1;
  return 0;
}
"""


def test_every_part_has_a_place_of_its_own(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "plan.cc").write_text("#include <algorithm>\n" + PROGRAM)
    binary = tmp_path / "plan"
    built = subprocess.run([compiler, "-O1", "-std=c++17", f"-I{CSRC}", str(tmp_path / "plan.cc"), "-o", str(binary)],
                           capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    done = subprocess.run([str(binary)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
