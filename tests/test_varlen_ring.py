"""The copies that the packed-prompt kernel waits for before a block gives its shared memory back: the device arithmetic of the
ring of K and V tiles restated, over any number of tiles asked for when the loads end or give up."""
import pytest

STAGES = 5


class Ring:
    def __init__(self):
        self.stage = self.round = 0

    def step(self):
        self.stage += 1
        if self.stage >= STAGES:
            self.stage, self.round = 0, self.round + 1

    def back(self):
        self.stage -= 1
        if self.stage < 0:
            self.stage, self.round = STAGES - 1, self.round - 1


@pytest.mark.parametrize("tiles", range(0, 4 * STAGES + 1))
def test_the_last_copy_into_every_buffer_is_waited_for(tiles):
    ring, last = Ring(), {}
    for _ in range(tiles):
        last[ring.stage] = ring.round              # the barrier's phase, whose parity the wait takes
        ring.step()
    waited = {}
    for _ in range(STAGES):
        if not (ring.round > 0 or ring.stage > 0):
            break
        ring.back()
        assert ring.stage not in waited
        waited[ring.stage] = ring.round
    assert waited == last


def test_a_step_back_undoes_a_step():
    ring = Ring()
    for i in range(1, 3 * STAGES):
        ring.step()
        ring.step()
        ring.back()
        assert ring.round * STAGES + ring.stage == i
