"""The paged cache through the C++ API (include/turboquant.h): exported, its
refusals without a GPU, and a run of its calls on one."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "gemma4metal_amd", "libturboquant_hip.so")
EXE = os.path.join(ROOT, "tests", "cpp", "test_paged")

CALLS = ["kv_append_int4_paged", "sdpa_int4_paged", "sdpa_int4_paged_prefill", "kv_pages_reserve", "kv_pages_fork",
         "kv_pages_free", "kv_pages_evict", "kv_pages_compact", "kv_pages_copy"]


def test_exported():
    out = subprocess.run(["nm", "-DC", "--defined-only", LIB], capture_output=True, text=True, check=True).stdout
    missing = [c for c in CALLS if f"turboquant::{c}(" not in out]
    assert not missing, missing


def test_refusals():
    r = subprocess.run([EXE, "refusals"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.count("PASS") == 15


@pytest.mark.gpu
def test_a_run_of_the_calls():
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.count("PASS") == 12


def test_calls_are_refused_by_their_own_checks():
    """By the check's message, with no GPU in sight: a missing check's GPU call fails
    otherwise."""
    env = {**os.environ, "HIP_VISIBLE_DEVICES": "", "ROCR_VISIBLE_DEVICES": ""}
    r = subprocess.run([os.path.join(ROOT, "tests", "cpp", "test_paged_calls"), "refusals"], capture_output=True, text=True,
                       timeout=60, env=env)
    assert r.returncode == 0 and r.stdout.count("PASS") == 35, r.stdout + r.stderr


def test_the_newer_calls_are_exported():
    out = subprocess.run(["nm", "-DC", "--defined-only", LIB], capture_output=True, text=True, check=True).stdout
    assert "turboquant::kv_pages_advance(" in out


@pytest.mark.gpu
def test_a_run_of_the_newer_calls():
    r = subprocess.run([os.path.join(ROOT, "tests", "cpp", "test_paged_calls")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.count("PASS") == 3, r.stdout + r.stderr
