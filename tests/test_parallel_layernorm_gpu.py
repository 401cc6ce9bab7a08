"""Two ranks with the layer-norm decoder, sharing GPU 0 over gloo (tests/test_parallel_gpu.py): its rows need no statistics of the other
rank's, in stage 1 by frames and by texels and in stage 2."""
import os
import sys

import pytest
import torch
import torch.multiprocessing as mp

from tests.test_parallel_gpu import FRAMES, ROOT, _free_port, _iterate

pytestmark = pytest.mark.gpu


def _build(batch_size, stage, bits8):
    from gaussianavatar_amd.avatar_model import AvatarModel, default_params
    mp_, npar, op = default_params(batch_size=batch_size, num_points=3000, query_posmap_size=64, inp_posmap_size=32 if stage == 1 else 64,
                                   image_width=96, image_height=96, num_frames=4, train_stage=stage, decoder_norm="layer", decoder_bits8=bits8)
    m = AvatarModel(mp_, npar, op, train=True)
    m.training_setup()
    if stage == 2:
        with torch.no_grad():                       # stand-in for the stage-1 checkpoint: ~1 cm Gaussians
            m.net.decoder.conv8N.bias.fill_(-4.0)
    return m, op


def _worker(rank, world, port, ret, mode, stage, bits8):
    sys.path.insert(0, ROOT)
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port),
                      HSA_ENABLE_IPC_MODE_LEGACY="0")
    from gaussianavatar_amd import parallel
    if mode:
        parallel.set_mode(mode)
    parallel.init_from_env(backend="gloo")
    torch.cuda.set_device(0)
    torch.manual_seed(1000 + rank)                  # replicas start different
    m, op = _build(2, stage, bits8)
    ret[rank] = _iterate(m, op, FRAMES[2 * rank:2 * rank + 2], stage=stage)
    parallel.barrier()
    torch.distributed.destroy_process_group()


@pytest.mark.parametrize("mode,stage,bits8", [("frames", 1, 0), ("texels", 1, 0), ("texels", 1, 1), (None, 2, 0)])
def test_two_ranks_equal_one_process_on_the_global_batch(mode, stage, bits8):
    """The bounds of test_parallel_gpu.py; with 8 bits a code next to a border goes the other way now and then, and the gradients are compared
    by norm, at the format's own rounding."""
    ret = mp.Manager().dict()
    mp.spawn(_worker, args=(2, _free_port(), ret, mode, stage, bits8), nprocs=2, join=True)
    r0, r1 = ret[0], ret[1]
    for a, b in zip(r0["grads"], r1["grads"]):
        assert float((a - b).abs().max()) <= 1e-6 * max(1.0, float(a.abs().max()))
    for a, b in zip(r0["params"], r1["params"]):
        assert float((a - b).abs().max()) <= 1e-6
    torch.manual_seed(1000)
    m, op = _build(4, stage, bits8)
    ref = _iterate(m, op, FRAMES, stage=stage)
    assert float((torch.cat([r0["image"], r1["image"]]) - ref["image"]).abs().mean()) <= 1e-5
    assert abs(r0["losses"][0] - ref["losses"][0]) <= 1e-5 * max(1.0, abs(ref["losses"][0]))
    gmax = max(float(g.abs().max()) for g in ref["grads"])
    for i, (a, b) in enumerate(zip(r0["grads"], ref["grads"])):
        if bits8:
            assert float((a - b).norm()) <= 2.0 ** -4 * float(b.norm()) + 2e-4 * gmax * b.numel() ** 0.5, i
        else:
            assert float((a - b).abs().max()) <= 2e-3 * float(b.abs().max()) + 2e-4 * gmax, i
