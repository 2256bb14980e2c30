"""Exercises the image decoder's steps for models of tokens in a sanitized build of the host library:
valid images, then hostile extents, slots and payloads, truncations and bit flips. Run by
tests/test_token_sanitizer_cpu.py in a child process; a report or a trap ends it."""
import itertools
import sys
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))

from synaptik_amd.program import ProgramBuilder  # noqa: E402
from tests import asan_driver  # noqa: E402  (loads the library that the first argument names)
from tests.test_token_model_gpu import SMALL, Model  # noqa: E402
from tests.test_token_steps_cpu import NAMES, built  # noqa: E402

HOSTILE = [-(1 << 63), -1, 0, 1, (1 << 31) - 1, 1 << 31, 1 << 40, 1 << 62, (1 << 63) - 200, (1 << 63) - 1]


def main():
    rng = np.random.default_rng(3)
    cases = 0
    for name in NAMES:
        assert asan_driver.validate(built(name).image()) == 0
        for i, j in itertools.combinations(range(9), 2):
            for a, b in itertools.product(HOSTILE, HOSTILE):
                pb = built(name)
                pb.steps[0].iargs[i], pb.steps[0].iargs[j] = a, b
                asan_driver.validate(pb.image())
                cases += 1
        for i in range(8):
            for slot in (-(1 << 31), -2, -1, 0, 1, 2, 3, 4, 5, 99, (1 << 31) - 1):
                pb = built(name)
                pb.steps[0].slots[i] = slot
                asan_driver.validate(pb.image())
                cases += 1
        for n in range(0, 24):
            pb = built(name)
            pb.steps[0].payload = bytes(rng.integers(0, 256, n, dtype=np.uint8))
            asan_driver.validate(pb.image())
            cases += 1
    pb = ProgramBuilder()
    Model(SMALL).build(pb)
    image = pb.image()
    assert asan_driver.validate(image) == 0
    for cut in rng.integers(0, len(image), 100):
        asan_driver.validate(image[:cut])
    for _ in range(2000):
        b = bytearray(image)
        for _ in range(int(rng.integers(1, 4))):
            b[int(rng.integers(0, len(b)))] ^= 1 << int(rng.integers(0, 8))
        asan_driver.validate(bytes(b))
        cases += 1
    print(f"images of token models ok: {cases} malformed cases", flush=True)


if __name__ == "__main__":
    main()
