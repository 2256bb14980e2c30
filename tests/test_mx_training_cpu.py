"""Programs with 8-bit checkpoints and microscaled weights, without a device: their schedules are
free of races, their memory is what the formats promise, and wrong arguments are refused."""
import itertools

import numpy as np
import pytest

from synaptik_amd.native import program_plan, validate_program_image
from synaptik_amd.training import (Adam, AdamW, GradientMode, MlpSpec, Sgd,
                                   encode_mx_weights, lower_forward, lower_mx_forward,
                                   lower_mx_weights, lower_training_step)
from tests import plan_hazards as H

SPECS = [([24, 32, 32, 5], "relu", "ce", 128), ([784, 1024, 1024, 10], "relu", "ce", 1024),
         ([16, 64, 1], "tanh", "mse", 256), ([4096] * 6, "relu", "mse", 4096),
         ([256, 512, 512, 512, 256], "sigmoid", "mse", 512), ([64, 48, 30], "tanh", "ce", 37),
         ([10, 7], None, "ce", 33)]
OPTS = [Sgd(0.05), Sgd(0.02, momentum=0.9, nesterov=True), Adam(1e-3), AdamW(1e-3)]
MODES = [(GradientMode.RESET_AND_STEP, False), (GradientMode.RESET_AND_STEP, True),
         (GradientMode.ACCUMULATE, False), (GradientMode.ACCUMULATE_AND_STEP, False)]


def mx_effects(st, stream=None, status_reads=True):
    """plan_hazards.effects with the microscaled steps, from what their kernels touch."""
    s = st.slots
    table = {17: ([0], [1, 2], False), 18: ([0, 1], [2], False), 19: ([0, 1, 2], [3, 4], True),
             20: ([0, 1, 2], [3], True), 21: ([0, 1, 2, 3], [4], True)}
    if st.opcode not in table:
        return PLAIN_EFFECTS(st, stream, status_reads)
    reads, writes, scratch = table[st.opcode]
    e = H.Effects()
    e.reads.update(("slot", s[i]) for i in reads if s[i] >= 0)
    e.writes.update(("slot", s[i]) for i in writes if s[i] >= 0)
    if scratch:
        H._scratch(e, ("scratch", stream))
    return e


PLAIN_EFFECTS = H.effects


@pytest.mark.parametrize("dims,act,loss,batch", SPECS, ids=str)
def test_checkpointed_steps_have_no_races(monkeypatch, dims, act, loss, batch):
    monkeypatch.setattr(H, "effects", mx_effects)
    spec = MlpSpec.chain(dims, hidden=act, loss=loss)
    for opt, (mode, clear), fmt in itertools.product(OPTS, MODES, ("e4m3", "e5m2")):
        pb, _ = lower_training_step(spec, batch, opt, mode=mode, clear_accumulator=clear, checkpoint=fmt)
        image = pb.image()
        validate_program_image(image)
        stream, wait, folded = program_plan(image)
        assert not H.check_plan(H.decode(image), stream, wait, folded)


def test_a_single_layer_needs_no_checkpoint():
    spec = MlpSpec.chain([10, 7], hidden=None, loss="mse")
    a, _ = lower_training_step(spec, 33, Sgd(0.1))
    b, _ = lower_training_step(spec, 33, Sgd(0.1), checkpoint="e4m3")
    assert a.image() == b.image()


def test_checkpoints_shrink_the_step():
    """Kept: 132 bytes a group of 128 values for each hidden layer, two activations, two cotangents
    and one weight gradient in binary32; beside them the scratch of the largest product."""
    n, layers = 1024, 24
    spec = MlpSpec.chain([n] * (layers + 1), hidden="relu")
    plain, _ = lower_training_step(spec, n, Sgd(0.1))
    kept, _ = lower_training_step(spec, n, Sgd(0.1), checkpoint="e4m3")
    plain, kept = validate_program_image(plain.image()), validate_program_image(kept.image())
    values = n * n
    fixed = (layers - 1) * (values // 128) * 132 + 6 * 4 * values
    scratch = (6 + 2 + 4 * 4) * values  # both operands' fragments and four partial sums
    assert fixed <= kept <= fixed + scratch + 64 * 1024 * layers
    assert kept < plain / 3


def test_wrong_arguments_are_refused():
    spec = MlpSpec.chain([8, 8, 8], hidden="relu")
    with pytest.raises(ValueError, match="checkpoint"):
        lower_training_step(spec, 4, Sgd(0.1), checkpoint="e2m1")
    with pytest.raises(ValueError, match="format"):
        lower_mx_forward(spec, 4, weights="int4")
    with pytest.raises(ValueError, match="per layer"):
        encode_mx_weights(None, spec, [np.zeros((8, 8))])

    class NoDevice:
        def upload(self, a):
            return a

    with pytest.raises(ValueError, match="shape"):
        encode_mx_weights(NoDevice(), spec, [np.zeros((8, 8)), np.zeros((8, 9))])


def test_output_activations_stay_refused():
    spec = MlpSpec.chain([8, 8, 8], hidden="relu", output="tanh")
    with pytest.raises(ValueError, match="identity"):
        lower_training_step(spec, 4, Sgd(0.1), checkpoint="e4m3")


def test_inference_programs_of_microscaled_weights():
    spec = MlpSpec.chain([617, 1021, 101], hidden="tanh")
    for batch in (1, 7, 300):
        for w, a in itertools.product(("e2m1", "e4m3", "e5m2"), repeat=2):
            pb = lower_mx_forward(spec, batch, weights=w, activations=a)
            validate_program_image(pb.image())
            assert pb.n_inputs == 2 * 2 + 2 + 1 and pb.n_outputs == 1
    validate_program_image(lower_mx_weights(spec, "e2m1").image())
    weights = sum(s.nbytes for s in lower_mx_forward(spec, 1).slots[:4])
    plain = sum(s.nbytes for s in lower_forward(spec, 1).slots[:2])
    assert weights < 0.15 * plain
