"""How paged attention deals its work, checked on the CPU over whole launches (tests/paged_deal_model.cpp runs the
arithmetic of torchvulkan_amd/csrc/paged_deal.h that the kernel runs)."""
import random
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    exe = tmp_path_factory.mktemp("deal") / "paged_deal_model"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", f"-I{ROOT / 'torchvulkan_amd' / 'csrc'}",
                    str(ROOT / "tests" / "paged_deal_model.cpp"), "-o", str(exe)], check=True)

    def run(bn=32, ct=1, resident=512, kvh=8, group=4, new=1, window=0, shared=0, batch=1, longest=1000, shortest=None, power=1):
        args = [bn, ct, resident, kvh, group, new, window, shared, batch, longest, longest if shortest is None else shortest, power]
        out = subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, timeout=120)
        assert out.returncode == 0, out.stderr
        word, launch, places = out.stdout.split()
        assert word == "ok"
        return int(launch), int(places)

    return run


# prompts and chunks of prompts whose launch has far more workgroups than there are stretches
@pytest.mark.parametrize("kw", [
    dict(ct=2, resident=256, kvh=8, group=4, new=42000, longest=42000),
    dict(ct=2, resident=256, kvh=8, group=8, new=28000, longest=28000),
    dict(ct=2, resident=512, kvh=4, group=4, new=100000, longest=100000),
    dict(ct=2, resident=256, kvh=8, group=4, new=2048, batch=30, longest=10500),
    dict(ct=2, resident=256, kvh=8, group=8, new=8192, batch=2, longest=65536),
])
@pytest.mark.parametrize("shared", [0, 1])
def test_long_prompts(model, kw, shared):
    launch, places = model(shared=shared, **kw)
    # scratch goes by the workgroups that run together, not by the launch
    assert launch > 4 * kw["resident"] and places <= 4 * kw["resident"]


@pytest.mark.parametrize("shared", [0, 1])
def test_a_few_long_among_many_short(model, shared):
    # most of the launch's workgroups have a segment to themselves, and no place in the scratch
    launch, places = model(ct=1, resident=256, kvh=8, batch=300, longest=3000, shortest=1, power=60, shared=shared)
    assert launch == 2400 + 512 and 0 < places <= 4 * 256


@pytest.mark.parametrize("bn", [16, 32])
@pytest.mark.parametrize("shared", [0, 1])
def test_sizes(model, bn, shared):
    rng = random.Random(1000 * bn + shared)
    for _ in range(150):
        batch = int(2 ** rng.uniform(0, 8))
        new = int(2 ** rng.uniform(0, rng.choice([0, 3, 12])))
        longest = max(new, int(2 ** rng.uniform(0, 17)))
        kvh, group = rng.choice([1, 2, 3, 8, 16]), rng.choice([1, 3, 4, 8, 16])
        # the model's time is that of its segments
        batch = max(1, min(batch, 60000 * 16 // (kvh * max(16, new * group)), (1 << 30) * 16 // (kvh * max(16, new * group) * longest)))
        model(bn=bn, ct=rng.choice([1, 2]), resident=256 * rng.randint(1, 4), kvh=kvh, group=group, new=new,
              window=rng.choice([0, 0, int(2 ** rng.uniform(0, 13))]), shared=shared, batch=batch, longest=longest,
              shortest=int(longest * rng.choice([1, 0.5, 0.02, 0])), power=rng.choice([1, 1, 4, 20]))
