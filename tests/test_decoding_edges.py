"""Decoding operators and generation at their edges: what can be checked without a GPU."""
import importlib
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import exploration_b200 as eb
from exploration_b200.ops.beam import select_reference

PAGED = Path(eb.__file__).parent / "csrc" / "paged"

# Runs the products of two softmax warpgroups in the issuer's order. At every wait of a warpgroup
# (it has seen the scores of its newest step and asked for that step's product or not yet) each
# number of finished products that is possible then is tried.
PHASES = r"""
#include <cstdio>
#include <vector>
#include "paged_phases.h"
using namespace eb::paged;

// mbarrier.try_wait.parity on a barrier with `phases` completed phases.
static bool passes(uint32_t phases, uint32_t parity) { return (phases & 1) != parity; }

// Completed phases of barrier b once `n` products of a warpgroup are complete.
static uint32_t phases_of(uint32_t b, uint32_t n, uint32_t barriers) { return n / barriers + (b < n % barriers); }

static long long wrong[2];
static void look(uint32_t wanted, uint32_t done) {
  const Phase p = product_phase(wanted);
  wrong[0] += passes(phases_of(p.barrier, done, kProductBarriers), p.parity) != (done > wanted);
  wrong[1] += passes(done, wanted & 1) != (done > wanted);      // one barrier a warpgroup
}

int main() {
  for (int bufs = 2; bufs <= 3; ++bufs) {
    uint32_t before[2] = {0, 0};           // products of earlier items (all complete)
    for (int round = 0; round < 64; ++round) {
      const int tiles = 1 + round % 7;
      const bool dual = (round / 7) % 2;
      const int steps = dual ? 2 * tiles : tiles;
      for (int i = 0; i < steps; ++i) {
        const int w = i & 1;
        // The scores of step i are issued after product i - bufs: products up to it are complete.
        uint32_t asked = 0, sure = 0;
        for (int j = w; j < i; j += 2) { ++asked; sure += j <= i - bufs; }
        if (asked > 0)                     // rescaling: waits for the product before this step's
          for (uint32_t n = sure; n <= asked; ++n) look(before[w] + asked - 1, before[w] + n);
        if (i + 2 >= steps)                // the item's end: waits for this step's product
          for (uint32_t n = sure; n <= asked + 1; ++n) look(before[w] + asked, before[w] + n);
      }
      for (int i = 0; i < steps; ++i) ++before[i & 1];
    }
  }
  std::printf("%lld %lld\n", wrong[0], wrong[1]);
}
"""


def run_host_program(tmp_path, text):
    """Compiles ``text`` against the kernels' host-checkable headers, runs it, returns its output's numbers."""
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    source, program = tmp_path / "check.cpp", tmp_path / "check"
    source.write_text(text)
    subprocess.run([compiler, "-std=c++17", "-O1", "-Wall", "-I", str(PAGED), str(source), "-o", str(program)],
                   check=True, timeout=120)
    done = subprocess.run([str(program)], check=True, capture_output=True, text=True, timeout=120)
    return [int(x) for x in done.stdout.split()]


def test_waits_for_products_are_never_ambiguous(tmp_path):
    """A wait for a warpgroup's product passes exactly when that product is complete."""
    wrong, wrong_with_one_barrier = run_host_program(tmp_path, PHASES)
    assert wrong == 0
    assert wrong_with_one_barrier > 0     # what the second barrier is for


def lowest_masked(dtype, vocab, spans):
    """Logits whose ``spans`` hold the type's lowest value, and one beam that holds nothing else."""
    logits = (3 * torch.randn(2, 3, vocab, generator=torch.Generator().manual_seed(vocab))).to(dtype)
    for lo, hi in spans:
        logits[:, :, lo:hi] = torch.finfo(dtype).min
    logits[1, 1] = torch.finfo(dtype).min
    return logits


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_with_the_types_lowest_value_as_a_mask(dtype):
    scores, ended = -torch.rand(2, 3).cumsum(1), torch.zeros(2, 3, dtype=torch.bool)
    for logits in (lowest_masked(dtype, 50, [(5, 20)]), lowest_masked(dtype, 50, [(2, 50)]),
                   (torch.randn(2, 3, 50) + 2.0 ** 20).to(dtype)):
        got = eb.beam_select(logits, scores, ended, -1)
        want = select_reference(logits.double(), scores, ended, -1)
        torch.testing.assert_close(got[0], want[0], atol=2e-5, rtol=0)
        assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))


EMPTY_POOLS = [(0, 12, 2, 16, 8), (2, 12, 0, 16, 8), (2, 12, 2, 16, 0)]     # no layers, no heads, no elements


def reorder_inputs(shape, device="cpu"):
    """Pools of ``shape`` and three beams, 21 tokens each, of which two take over the second one's state."""
    k, v = torch.zeros(shape, device=device), torch.zeros(shape, device=device)
    tables = torch.arange(9, dtype=torch.int32, device=device).view(1, 3, 3)
    spare = torch.arange(9, 12, dtype=torch.int32, device=device).view(1, 3)
    return k, v, tables, spare, torch.tensor([[1, 1, 1]], device=device), \
        torch.tensor([21], dtype=torch.int32, device=device)


REORDERED = [[[3, 9, 2], [3, 4, 5], [3, 11, 8]]], [[1, 10, 7]]


@pytest.mark.parametrize("shape", EMPTY_POOLS)
def test_reorder_of_empty_pools(shape):
    fresh, freed = eb.beam_reorder(*reorder_inputs(shape))
    assert (fresh.tolist(), freed.tolist()) == REORDERED


def test_reorder_refuses_pages_without_tokens():
    with pytest.raises(ValueError, match="at least one token"):
        eb.beam_reorder(*reorder_inputs((2, 12, 2, 0, 8)))


# Keys and values go out in turn, tile by tile; a producer that gives up after any number of copies waits
# for all that may be under way: the newest `stages` of each operand, each wait passing only once that copy
# has landed (the one before it in its slot has, or the slot would not have been reused).
COPIES = r"""
#include <cstdio>
#include "paged_phases.h"
using namespace eb::paged;

int main() {
  long long wrong = 0, cases = 0;
  for (uint32_t stages = 2; stages <= 4; stages += 2)
    for (uint32_t copies = 0; copies < 40; ++copies) {
      CopyRing rings[2];
      for (uint32_t i = 0; i < copies; ++i) {
        CopyRing& ring = rings[i & 1];
        const Phase slot = ring.next(stages);
        wrong += slot.barrier != ring.issued % stages || ring.reuses(stages) != (ring.issued >= stages);
        ++ring.issued;
      }
      for (int part = 0; part < 2; ++part) {
        const uint32_t issued = (copies + 1 - part) / 2;
        wrong += rings[part].issued != issued;
        uint32_t n = issued > stages ? issued - stages : 0;
        rings[part].drain(stages, [&](uint32_t slot, uint32_t parity) {
          const uint32_t before = n / stages;        // phases of the slot's barrier without copy n
          wrong += slot != n % stages || (before & 1) != parity || ((before + 1) & 1) == parity;
          ++n;
          ++cases;
        });
        wrong += n != issued;
      }
    }
  std::printf("%lld %lld\n", wrong, cases);
}
"""


def test_a_producer_that_gives_up_waits_for_every_copy(tmp_path):
    wrong, waits = run_host_program(tmp_path, COPIES)
    assert wrong == 0 and waits > 100


def test_generate_raises_when_a_kernel_gave_up_a_wait(monkeypatch):
    generation = importlib.import_module("exploration_b200.runtime.generate")
    torch.manual_seed(0)
    model, looked = eb.BaselineModel(19, dim=32, heads=4, layers=1).eval(), []
    monkeypatch.setattr(generation, "check_waits", looked.append)
    eb.generate(model, [[1, 2], [3]], 3, page=16)
    assert looked == [torch.device("cpu")]
    monkeypatch.undo()

    # The error word of a device, read and cleared: (site, CTA).
    words = {1: [(2, 37), (0, 0)]}
    order = []

    class Extension:
        def device_errors(self, index):
            order.append("read")
            return words[index].pop(0)

    class Stream:
        def synchronize(self):
            order.append("synchronize")

    monkeypatch.setattr(generation._native, "load", lambda: Extension())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: Stream())
    with pytest.raises(RuntimeError, match="site 2, CTA 37"):
        generation.check_waits(torch.device("cuda", 1))
    generation.check_waits(torch.device("cuda", 1))
    generation.check_waits(torch.device("cpu"))
    assert order == ["synchronize", "read"] * 2


@pytest.mark.parametrize("prompt", [[1, 19], [-1], torch.tensor([3, 400])])
def test_generate_refuses_tokens_outside_the_vocabulary(prompt):
    torch.manual_seed(0)
    model = eb.BaselineModel(19, dim=32, heads=4, layers=1).eval()
    eb.generate(model, [[0, 18]], 1, page=16)
    with pytest.raises(ValueError, match="vocabulary"):
        eb.generate(model, [[1], prompt], 1, page=16)


def decoding_calls(device="cpu"):
    """Every decoding operator with the names of its differentiable inputs."""
    def new(*shape):
        return torch.randn(*shape, device=device)

    tables, positions = (torch.zeros(1, n, dtype=torch.int32, device=device) for n in (1, 2))
    paged = {"q": new(1, 2, 4, 8), "k": new(1, 2, 2, 8), "v": new(1, 2, 2, 8), "cos": new(20, 4), "sin": new(20, 4),
             "k_cache": new(3, 2, 16, 8), "v_cache": new(3, 2, 16, 8)}
    attention = {n: paged[n].clone() for n in ("q", "k_cache", "v_cache")}
    select = {"logits": new(2, 3, 5), "scores": new(2, 3)}
    ended = torch.zeros(2, 3, dtype=torch.bool, device=device)
    k, v, *rest = reorder_inputs((2, 12, 2, 16, 8), device)
    return [
        (lambda **x: eb.paged_append(*x.values(), tables, positions), paged),
        (lambda **x: eb.paged_attention(*x.values(), tables, positions), attention),
        (lambda **x: eb.beam_select(*x.values(), ended, 1), select),
        (lambda **x: eb.beam_reorder(*x.values(), *rest), {"k_cache": k, "v_cache": v}),
    ]


def check_gradients_are_refused(device):
    from torch.autograd import forward_ad
    for call, inputs in decoding_calls(device):
        call(**inputs)
        for name, x in inputs.items():
            leaf = x.clone().requires_grad_()
            with pytest.raises(ValueError, match="no gradient"):
                call(**{**inputs, name: leaf})
            with torch.no_grad():
                call(**{**inputs, name: leaf})
                with forward_ad.dual_level():
                    with pytest.raises(ValueError, match="no gradient"):
                        call(**{**inputs, name: forward_ad.make_dual(x.clone(), torch.ones_like(x))})
                    call(**inputs)


def test_gradients_and_tangents_are_refused():
    check_gradients_are_refused("cpu")
