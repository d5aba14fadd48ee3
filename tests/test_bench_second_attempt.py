"""The second attempt of a rank whose captured step hangs or cannot be used (bench.py): a child process that ends when the rank's own process ends, on the CPU
(the rehearsed attempt is the launch check over gloo)."""
import os
import signal
import subprocess
import sys
import time

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _rank(body, world, **env):
    """a process that arms the watchdog and goes on with `body`; its second attempt is `bench.py --dry-run-launch --gpus world` as rank 0"""
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    env = dict({k: v for k, v in os.environ.items() if not k.startswith(("TORCHELASTIC", "DH_BENCH"))}, RANK="0", LOCAL_RANK="0", WORLD_SIZE=str(world),
               MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), DH_DIST_BACKEND="gloo", **env)
    code = "import sys, time; sys.path.insert(0, %r); import bench; sys.argv = ['bench.py', '--dry-run-launch', '--gpus', '%d', '--graph', '1']\n%s" % (ROOT, world, body)
    p = subprocess.Popen([sys.executable, "-u", "-c", code], env=env, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, cwd=ROOT)
    p.port = port + 1                                # where its second attempt listens
    return p


def _children(pid):
    out = []
    for t in os.listdir("/proc/%d/task" % pid):
        with open("/proc/%d/task/%s/children" % (pid, t)) as f:
            out += [int(c) for c in f.read().split()]
    return out


def _alive(pid):
    try:
        with open("/proc/%d/stat" % pid) as f:
            return f.read().rsplit(")", 1)[1].split()[0] != "Z"
    except OSError:
        return False


def _wait(what, seconds=60):
    end = time.time() + seconds
    while time.time() < end:
        v = what()
        if v:
            return v
        time.sleep(0.1)
    return what()


def test_the_second_attempt_speaks_for_the_rank():
    p = _rank("bench._arm_watchdog(0.1, 'a step')\ntime.sleep(600)", 1)
    out, err = p.communicate(timeout=120)
    assert p.returncode == 0 and '"dry_run": true' in out and "watchdog: a step made no progress" in err, err[-2000:]


@pytest.mark.parametrize("sig", [signal.SIGTERM, signal.SIGKILL])
@pytest.mark.parametrize("ready", [False, True])
def test_the_second_attempt_ends_with_its_rank(sig, ready):
    """a launcher that terminates or kills the rank knows one process: the attempt under way (here it waits for a rank 1 that never comes) goes with it"""
    p, kids = _rank("bench._arm_watchdog(0.1, 'a step')\ntime.sleep(600)", 2), []
    try:
        kids = _wait(lambda: _children(p.pid))
        assert len(kids) == 1
        if ready:                                    # (it listens for its peers: up and running)
            assert _wait(lambda: any(line.split()[1].endswith(":%04X" % p.port) and line.split()[3] == "0A" for t in ("tcp", "tcp6") for line in open("/proc/net/" + t).readlines()[1:]))
        p.send_signal(sig)
        p.wait(30)
        assert _wait(lambda: not _alive(kids[0]), 60), "the second attempt outlived its rank"
    finally:
        for pid in [p.pid] + kids:
            try:
                os.kill(pid, signal.SIGKILL)
            except OSError:
                pass
        p.communicate()


@pytest.mark.parametrize("late", ["pass", "raise ValueError('the step came to nothing')", "[w.check() for w in [W]]; print('went on')"])
def test_a_step_that_comes_back_too_late_says_nothing_more(late):
    """the step returns, raises or begins the next one while the second attempt runs: the attempt's line and exit code are the rank's"""
    p = _rank("W = bench._arm_watchdog(0.1, 'a step')\ndef late():\n    time.sleep(1.0)\n    %s\nW.guard(late)\nprint('went on')" % late, 1)
    out, err = p.communicate(timeout=120)
    assert p.returncode == 0 and '"dry_run": true' in out and "went on" not in out and "ValueError" not in err, (out, err[-2000:])


def test_a_step_in_time_disarms_the_watchdog():
    p = _rank("W = bench._arm_watchdog(0.5, 'a step')\nW.guard(lambda: None)\nW._fire()\ntime.sleep(1.0)\nW.check()\nprint('went on')", 1)
    out, err = p.communicate(timeout=120)
    assert p.returncode == 0 and out.strip() == "went on" and "watchdog" not in err
    p = _rank("W = bench._arm_watchdog(0.5, 'a step')\ndef bad():\n    raise ValueError('of its own')\nW.guard(bad)", 1)
    out, err = p.communicate(timeout=120)
    assert p.returncode == 1 and "of its own" in err and "watchdog" not in err


def test_an_unusable_step_starts_over():
    p = _rank("W = bench._arm_watchdog(60, 'a step')\nW.cancel()\nW.start_over('no capture')\nprint('went on')", 1)
    out, err = p.communicate(timeout=120)
    assert p.returncode == 0 and '"dry_run": true' in out and "went on" not in out and "captured step unusable (no capture)" in err


def test_an_attempt_that_fails_fails_the_rank():
    p = _rank("sys.argv += ['--gpus', '2']\nbench._arm_watchdog(0.1, 'a step')\ntime.sleep(600)", 1)     # (its world is 1)
    out, err = p.communicate(timeout=120)
    assert p.returncode == 3, err[-2000:]
