"""The layer entry points' host side under AddressSanitizer + UndefinedBehaviorSanitizer: tests/host/layer_argument_checks.cpp, built with
the library by `make asan`, walks their refusals and no-ops and sizes workspaces over the whole range of shapes.  It needs no GPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_layer_argument_checks_under_asan_and_ubsan():
    csrc = os.path.join(ROOT, 'nerf_amd', 'csrc')
    subprocess.check_call(['make', '-C', csrc, '-j8', 'asan'], stdout=subprocess.DEVNULL)      # up to date after build()
    exe = os.path.join(ROOT, 'nerf_amd', 'lib', 'layer_argument_checks_asan')
    env = dict(os.environ, ASAN_OPTIONS='detect_leaks=0:abort_on_error=0', UBSAN_OPTIONS='print_stacktrace=1')
    r = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, env=env, timeout=300)
    out = r.stdout.decode(errors='replace')
    assert r.returncode == 0, out[-4000:]
    assert 'all layer argument checks passed' in out and 'runtime error' not in out and 'AddressSanitizer' not in out, out[-4000:]
