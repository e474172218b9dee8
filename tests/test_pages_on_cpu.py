"""Runs tests/cpp/test_pages_on_cpu.cpp: the page kernels themselves, compiled
for the host over a lock-step lane emulation, on random lives of a cache (with lists
that name sequences twice, out of range, beyond what fits) against a book kept
one entry at a time, on copies between pools, and on books and lists of random words,
which may not make them touch anything outside."""
import os
import subprocess

SHARDS = 4


def test_pages_follow_the_book_and_touch_nothing_else(pkg):
    exe = pkg.build.PAGES_ON_CPU_TEST
    if not os.path.exists(exe):
        pkg.build.build_pages_on_cpu_test()
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1")
    procs = [subprocess.Popen([exe, "--shard", "%d/%d" % (i, SHARDS)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                              text=True, env=env) for i in range(SHARDS)]
    for i, proc in enumerate(procs):
        out, _ = proc.communicate(timeout=1200)
        assert proc.returncode == 0, "shard %d:\n%s" % (i, out[-4000:])
        assert out.strip().endswith("0 failures"), out[-2000:]
