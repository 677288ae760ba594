"""Which form of its kernel each call of the sequence operators takes: the library's own rules (turboae_seq_plan.hpp), compiled for the host."""
import os
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <stdio.h>
#include <string.h>
#include "turboae_seq_plan.hpp"
using namespace tae::seq;
int main() {
    char op[16];
    long long v[5];
    while (scanf("%15s %lld %lld %lld %lld %lld", op, v, v + 1, v + 2, v + 3, v + 4) == 6) {
        if (!strcmp(op, "scan")) {                       // dtype batch len channels states -> lanes per_lane pieces step_sequences state_lanes
            tae_scan_args a = {};
            a.dtype = (int)v[0], a.batch = (int)v[1], a.len = (int)v[2], a.channels = (int)v[3], a.states = (int)v[4];
            ScanPlan s;
            const bool ok = plan_scan(&a, &s);
            const int V = a.states % 4 ? 1 : 4;
            printf("%d %d %d %d %d %d\n", ok, s.lanes, s.per_lane, s.pieces, step_sequences(a.batch, a.channels, a.states, V), state_lanes(a.states, V));
        } else if (!strcmp(op, "int8")) {                // dtype rows inputs outputs - -> form
            tae_int8_args a = {};
            a.dtype = (int)v[0], a.rows = (int)v[1], a.inputs = (int)v[2], a.outputs = (int)v[3];
            printf("%d %d\n", int8_sizes(&a), (int)int8_form(&a));
        } else {                                         // dtype rows vocab top aligned -> lanes elements parts
            tae_logprobs_args a = {};
            a.dtype = (int)v[0], a.rows = (int)v[1], a.vocab = (int)v[2], a.top = (int)v[3];
            LogprobsPlan s;
            const bool ok = plan_logprobs(&a, v[4] != 0, &s);
            printf("%d %d %d %d\n", ok, s.lanes, s.ept, s.parts);
        }
    }
    return 0;
}
"""

DTYPE = {"f32": 0, "f16": 1, "bf16": 2}
TILES = ((4, 1), (8, 1), (16, 1), (8, 2), (16, 2), (8, 4), (16, 4))          # lanes for a channel, states of each
INT8_FORMS = ["rows", "few16", "few32", "few64", "tiles128", "tiles128_two", "tiles256"]


def compiler():
    return shutil.which("g++") or shutil.which("c++")


class Forms:
    def __init__(self, folder):
        src, self.exe = os.path.join(folder, "forms.cpp"), os.path.join(folder, "forms")
        with open(src, "w") as fh:
            fh.write(PROGRAM)
        subprocess.check_call([compiler(), "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "turboae_amd", "csrc"), src, "-o", self.exe])

    def ask(self, lines):
        out = subprocess.run([self.exe], input="\n".join(" ".join(str(v) for v in line) for line in lines) + "\n", capture_output=True, text=True, timeout=60, check=True).stdout
        answers = [[int(v) for v in line.split()] for line in out.splitlines()]
        assert len(answers) == len(lines) and all(a[0] == 1 for a in answers)
        return [a[1:] for a in answers]

    def scan(self, cases):
        """(dtype, batch, len, channels, states) -> the kernel with its template arguments"""
        found = []
        for (dt, B, L, E, N), (lanes, per_lane, pieces, each, share) in zip(cases, self.ask([("scan", DTYPE[c[0]], *c[1:]) for c in cases])):
            V = 1 if N % 4 else 4
            if L == 1:
                found.append(("step", V, share, each))
            elif lanes == 0:
                found.append(("short", V, share))
            else:
                found.append(("lane", N == 16, pieces > 1) if lanes == 1 else ("tile", lanes, per_lane, pieces > 1, 1 if E % 4 else 4))
        return found

    def int8(self, cases):
        """(dtype, rows, inputs, outputs) -> name of the form"""
        return [INT8_FORMS[a[0]] for a in self.ask([("int8", DTYPE[c[0]], *c[1:], 0) for c in cases])]

    def logprobs(self, cases):
        """(dtype, rows, vocab, top, rows on 16-byte boundaries) -> (lanes, elements of a lane, parts)"""
        return [tuple(a) for a in self.ask([("logp", DTYPE[c[0]], *c[1:4], int(c[4])) for c in cases])]
