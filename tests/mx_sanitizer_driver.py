"""Exercises the image decoder's microscaled steps in a sanitized build of the host library: valid
images of every step and lowering, then one and two hostile extents, hostile slots, truncations and
bit flips. Run by tests/test_mx_sanitizer_cpu.py in a child process; a report or a trap ends it."""
import itertools
import sys
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))

from tests import asan_driver  # noqa: E402  (loads the library that the first argument names)
from synaptik_amd.training import (Adam, GradientMode, MlpSpec, Sgd, lower_mx_forward,  # noqa: E402
                                   lower_mx_weights, lower_training_step)
from tests.test_mx_cpu import NAMES, built  # noqa: E402

HOSTILE = [-(1 << 63), -1, 0, 1, (1 << 31) - 1, 1 << 31, (1 << 31) + 200, 1 << 40, 1 << 62, (1 << 63) - 200,
           (1 << 63) - 1]


def main():
    rng = np.random.default_rng(3)
    cases = 0
    for name in NAMES:
        assert asan_driver.validate(built(name).image()) == 0
        args = len(built(name).steps[0].iargs)
        for i, j in itertools.combinations(range(args), 2):
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
    spec = MlpSpec.chain([40, 70, 33, 6], hidden="tanh", loss="ce")
    images = [lower_mx_weights(spec).image(), lower_mx_forward(spec, 9).image()]
    for opt, mode in itertools.product((Sgd(0.1, momentum=0.9), Adam(1e-3)),
                                       (GradientMode.RESET_AND_STEP, GradientMode.ACCUMULATE,
                                        GradientMode.ACCUMULATE_AND_STEP)):
        images.append(lower_training_step(spec, 64, opt, mode=mode, checkpoint="e5m2")[0].image())
    for image in images:
        assert asan_driver.validate(image) == 0
        for cut in rng.integers(0, len(image), 60):
            asan_driver.validate(image[:cut])
        for _ in range(400):
            b = bytearray(image)
            for _ in range(int(rng.integers(1, 4))):
                b[int(rng.integers(0, len(b)))] ^= 1 << int(rng.integers(0, 8))
            asan_driver.validate(bytes(b))
            cases += 1
    print(f"microscaled images ok: {cases} malformed cases", flush=True)


if __name__ == "__main__":
    main()
