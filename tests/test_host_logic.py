"""CPU tests of the host-side logic: packed-layout bookkeeping, column maps, config / state-dict compatibility with the
reference, dotted-path aliases for YAML configs, and the N > 1 gradient exchange (gloo, world_size 2)."""
import json
import os
import subprocess
import sys
import textwrap

import pytest
import torch
import yaml

from conftest import ROOT, load_golden


def test_colmaps_are_permutations():
    from presight_amd.field_ops import colour_colmap
    from presight_amd.ops import chain_colmap, linear_colmap

    for n in (8, 32, 40, 47, 64):
        ks = (n + 3) // 4
        cm = [c for c in linear_colmap(ks, n) if c >= 0]
        assert sorted(cm) == list(range(n))
    for n in (16, 32, 64, 80):
        cm = [c for c in chain_colmap(n // 4, n) if c >= 0]
        assert sorted(cm) == list(range(n))
    for a in (0, 4, 16):
        cm = [c for c in colour_colmap(a) if c >= 0]
        assert sorted(cm) == list(range(31 + a))  # SH16 + geo15 + app


def test_model_state_dict_matches_reference_checkpoint_keys(gold_model):
    """Every parameter key of the reference's (torch-implementation) NerfactoNuscMSModel exists with the same shape."""
    from conftest import model_fixture_setup
    from presight_amd.model import NerfactoNuscMSModel, NerfactoNuscMSModelConfig

    cfg, scene, P, _ = model_fixture_setup(gold_model)
    m = cfg["main"]
    conf = NerfactoNuscMSModelConfig(
        hidden_dim=m["hidden_dim"], hidden_dim_color=m["hidden_dim_color"], num_levels=m["num_levels"], max_res=m["max_res"],
        log2_hashmap_size=m["log2_hashmap_size"], features_per_level=m["features_per_level"], use_lidar_loss=False,
        proposal_net_args_list=[dict(features_per_level=p["features_per_level"], log2_hashmap_size=p["log2_hashmap_size"],
                                     num_levels=p["num_levels"], base_res=p["base_res"], max_res=p["max_res"],
                                     hidden_dim=p["hidden_dim"], use_linear=False) for p in cfg["props"]])
    model = NerfactoNuscMSModel(conf, num_train_cameras=cfg["num_cameras"], num_train_videos=cfg["num_videos"], dino_to_rgb=None,
                                centroids=scene["centroids"], aabbs=scene["aabbs"])
    sd = model.state_dict()
    for k, v in P.items():
        assert k in sd and tuple(sd[k].shape) == tuple(v.shape), k
    # the reference aliases mlp_base = Sequential(grid, mlp): those duplicate keys exist too
    assert "field.fields.0.mlp_base.0.hash_table" in sd and "proposal_networks.0.fields.0.mlp_base.1.layers.0.weight" in sd
    assert set(model.get_param_groups()) == {"proposal_networks", "fields"}


def test_yaml_config_with_reference_dotted_path_loads():
    from presight_amd import compat

    compat.install()
    text = textwrap.dedent("""
        !!python/object:nerfstudio.models.PreSight.nerfacto_nusc_ms.NerfactoNuscMSModelConfig
        near_plane: 0.005
        far_plane: 50.0
        piecewise_sampler_threshold: 5.0
        num_levels: 10
        features_per_level: 4
        log2_hashmap_size: 20
        max_res: 16384
        use_lidar_loss: false
        implementation: tcnn+fp32
        num_proposal_samples_per_ray: !!python/tuple [128, 64]
        pulse_width: !!python/tuple [0.03, 0.003]
    """)
    conf = yaml.load(text, Loader=yaml.Loader)
    from presight_amd.model import NerfactoNuscMSModelConfig

    assert isinstance(conf, NerfactoNuscMSModelConfig)
    assert conf.far_plane == 50.0 and conf.num_levels == 10 and conf.implementation == "tcnn+fp32"
    import nerfstudio.fields.PreSight.ingp_field as ref_path

    assert hasattr(ref_path, "iNGPField")


def test_anneal_and_update_schedule_match_reference_formulas():
    """SURVEY Appendix A.7."""
    import numpy as np

    from presight_amd.model import NerfactoNuscMSModel, NerfactoNuscMSModelConfig

    conf = NerfactoNuscMSModelConfig(use_lidar_loss=False, num_levels=2, features_per_level=2, log2_hashmap_size=4, max_res=64,
                                     hidden_dim=32, hidden_dim_color=32, proposal_weights_anneal_max_num_iters=1000,
                                     proposal_net_args_list=[dict(features_per_level=1, log2_hashmap_size=4, num_levels=2,
                                                                  base_res=16, max_res=32, hidden_dim=32, use_linear=False)])
    m = NerfactoNuscMSModel(conf, num_train_cameras=2, num_train_videos=1, dino_to_rgb=None, centroids=torch.zeros(1, 3),
                            aabbs=torch.tensor([[[-1.0, -1, -1], [1, 1, 1]]]))
    for step in (0, 100, 500, 1000, 5000):
        x = np.clip(step / 1000, 0, 1)
        assert abs(m.anneal_for_step(step) - 10 * x / (9 * x + 1)) < 1e-12
    s = m.proposal_sampler
    assert s.update_sched(0) == 1 and s.update_sched(500) == 2.5 and s.update_sched(5000) == 5


def test_spaced_sampler_takes_the_reference_callables():
    """ns/models/PreSight/nerfacto_nusc_ms.py:311-316 constructs SpacedSampler(spacing_fn=..., spacing_fn_inv=..., single_jitter=...):
    the threshold is recovered from the callables; a spacing that the kernels do not implement is rejected, never ignored."""
    from presight_amd.samplers import SpacedSampler, piecewise_threshold_of

    for thr in (1.0, 5.0, 2.5):
        s = SpacedSampler(spacing_fn=lambda x: torch.where(x < thr, x / (2 * thr), 1 - 1 / (2 * x / thr)),
                          spacing_fn_inv=lambda x: torch.where(x < 0.5, x * (2 * thr), thr / (2 - 2 * x)), single_jitter=True)
        assert s.thr == thr
    assert SpacedSampler(piecewise_threshold=5.0, single_jitter=True).thr == 5.0
    with pytest.raises(NotImplementedError):
        SpacedSampler(spacing_fn=lambda x: x, spacing_fn_inv=lambda x: x, single_jitter=True)  # UniformSampler's spacing
    with pytest.raises(NotImplementedError):
        SpacedSampler(spacing_fn=lambda x: torch.log(1 + x), spacing_fn_inv=lambda x: torch.exp(x) - 1, single_jitter=True)
    with pytest.raises(NotImplementedError):  # right spacing, wrong inverse
        SpacedSampler(spacing_fn=lambda x: torch.where(x < 5.0, x / 10.0, 1 - 1 / (2 * x / 5.0)), spacing_fn_inv=lambda x: x * 10.0,
                      single_jitter=True)
    with pytest.raises(ValueError):
        SpacedSampler(spacing_fn=lambda x: torch.where(x < 5.0, x / 10.0, 1 - 1 / (2 * x / 5.0)), single_jitter=True, piecewise_threshold=1.0)
    with pytest.raises(ValueError):
        SpacedSampler(single_jitter=True)
    assert piecewise_threshold_of(lambda x: torch.where(x < 0.7, x / 1.4, 1 - 0.7 / (2 * x))) == 0.7


def test_model_through_the_reference_call_sequence():
    """What the reference's pipeline / trainer do with a model (ns/pipelines/PreSight/my_pipeline.py:107-118, ns/engine/
    trainer.py:154-160,252-267): config.setup(**kwargs) -> get_param_groups -> get_training_callbacks(attributes) -> callbacks
    run before / after every iteration -> get_image_metrics_and_images on a rendered image.  YAML round trip included."""
    import numpy as np

    from presight_amd import compat

    compat.install()
    from nerfstudio.engine.callbacks import TrainingCallback, TrainingCallbackAttributes, TrainingCallbackLocation
    from nerfstudio.models.PreSight.nerfacto_nusc_ms import NerfactoNuscMSModel, NerfactoNuscMSModelConfig

    conf = NerfactoNuscMSModelConfig(use_lidar_loss=False, num_levels=2, features_per_level=2, log2_hashmap_size=4, max_res=64,
                                     hidden_dim=32, hidden_dim_color=32, proposal_weights_anneal_max_num_iters=1000,
                                     piecewise_sampler_threshold=5.0,
                                     proposal_net_args_list=[dict(features_per_level=1, log2_hashmap_size=4, num_levels=2,
                                                                  base_res=16, max_res=32, hidden_dim=32, use_linear=False)])
    conf = yaml.load(yaml.dump(conf), Loader=yaml.Loader)  # what ns-train writes to config.yml and eval_setup reads back
    assert isinstance(conf, NerfactoNuscMSModelConfig) and conf.piecewise_sampler_threshold == 5.0
    model = conf.setup(scene_box=None, num_train_data=-1, num_train_cameras=2, num_train_videos=1, dino_to_rgb=None,
                       centroids=torch.zeros(1, 3), aabbs=torch.tensor([[[-1.0, -1, -1], [1, 1, 1]]]))
    assert isinstance(model, NerfactoNuscMSModel)
    assert model.proposal_sampler.initial_sampler.thr == 5.0  # recovered from the two lambdas of nerfacto_nusc_ms.py:311-316
    assert set(model.get_param_groups()) == {"proposal_networks", "fields"}
    cbs = model.get_training_callbacks(TrainingCallbackAttributes(optimizers=None, grad_scaler=None, pipeline=None))
    assert len(cbs) == 2 and all(isinstance(c, TrainingCallback) for c in cbs)
    assert cbs[0].where_to_run == [TrainingCallbackLocation.BEFORE_TRAIN_ITERATION]
    assert cbs[1].where_to_run == [TrainingCallbackLocation.AFTER_TRAIN_ITERATION]
    for step in (0, 1, 2, 250):
        for cb in cbs:
            cb.run_callback_at_location(step, TrainingCallbackLocation.BEFORE_TRAIN_ITERATION)
        x = np.clip(step / 1000, 0, 1)
        assert model.step == step and abs(model.proposal_sampler._anneal - 10 * x / (9 * x + 1)) < 1e-12
        before = model.proposal_sampler._steps_since_update
        for cb in cbs:
            cb.run_callback_at_location(step, TrainingCallbackLocation.AFTER_TRAIN_ITERATION)
        assert model.proposal_sampler._step == step and model.proposal_sampler._steps_since_update == before + 1
    conf2 = NerfactoNuscMSModelConfig(use_lidar_loss=False, use_proposal_weight_anneal=False, num_levels=2, features_per_level=2,
                                      log2_hashmap_size=4, max_res=64, hidden_dim=32, hidden_dim_color=32,
                                      proposal_net_args_list=conf.proposal_net_args_list)
    m2 = conf2.setup(num_train_cameras=2, num_train_videos=1, dino_to_rgb=None, centroids=torch.zeros(1, 3),
                     aabbs=torch.tensor([[[-1.0, -1, -1], [1, 1, 1]]]))
    assert m2.get_training_callbacks(None) == []  # nerfacto_nusc_ms.py:421: both callbacks hang on use_proposal_weight_anneal
    with pytest.raises(AssertionError):
        TrainingCallback([TrainingCallbackLocation.AFTER_TRAIN], func=lambda s: None)  # callbacks.py:79-81: needs a `step` argument
    # evaluation image -> metrics + images (nerfacto_nusc_ms.py:647-686)
    H, W = 6, 8
    g = torch.Generator().manual_seed(0)
    outputs = {"rgb": torch.rand(H, W, 3, generator=g), "accumulation": torch.rand(H, W, 1, generator=g), "depth": torch.rand(H, W, 1, generator=g) * 9,
               "prop_depth_0": torch.rand(H, W, 1, generator=g), "prop_depth_1": torch.rand(H, W, 1, generator=g)}
    batch = {"rgb": torch.rand(H, W, 3, generator=g)}
    metrics, images = model.get_image_metrics_and_images(outputs, batch)
    mse = float(((outputs["rgb"] - batch["rgb"]) ** 2).mean())
    assert abs(metrics["psnr"] - 10 * np.log10(1 / mse)) < 1e-4
    assert images["img"].shape == (H, 2 * W, 3) and torch.equal(images["img"][:, :W], batch["rgb"]) and torch.equal(images["img"][:, W:], outputs["rgb"])
    assert set(images) == {"img", "accumulation", "depth", "prop_depth_0", "prop_depth_1"}
    for k in ("accumulation", "depth", "prop_depth_0"):
        assert images[k].shape == (H, W, 3) and float(images[k].min()) >= 0 and float(images[k].max()) <= 1


_WORKER = textwrap.dedent("""
    import os, sys, torch, torch.distributed as dist
    sys.path.insert(0, {root!r})
    from presight_amd.dist import FlatGrads, init_from_env
    rank, local, world = init_from_env("cpu")
    torch.manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(5, 3)), torch.nn.Parameter(torch.randn(7)), torch.nn.Parameter(torch.randn(2, 2, 2))]
    fg = FlatGrads(params)
    for i, p in enumerate(params):
        (p * (rank + 1) * (i + 1)).sum().backward()
    assert all(p.grad.data_ptr() >= fg.flat.data_ptr() for p in params)  # grads are views of the flat buffer
    fg.all_reduce_mean()
    expect = [(1 + 2) / 2 * (i + 1) for i in range(3)]
    for p, e in zip(params, expect):
        assert torch.allclose(p.grad, torch.full_like(p, e)), (rank, p.grad, e)
    # "unused parameter" case: rank 1 contributes nothing for params[1]
    fg.zero_()
    if rank == 0:
        (params[1] * 4).sum().backward()
    fg.all_reduce_mean()
    assert torch.allclose(params[1].grad, torch.full_like(params[1], 2.0))
    # "received a gradient this step" flags: local by default, OR-ed over ranks on request (DDP semantics for routing)
    assert fg.touched() == [False, rank == 0, False]
    fg.flags_may_differ_across_ranks = True
    assert fg.touched() == [False, True, False]
    assert fg.touched_ranges() == [(16, 24)]  # 15 floats padded to 16, then 7 padded to 8
    # bucketed exchange launched from the gradient hooks: bucket 0 = params[0:2], bucket 1 = params[2:3]
    fg.flags_may_differ_across_ranks = False
    fg.enable_overlap([params[0:2], params[2:3]])
    fg.zero_()
    for i, p in enumerate(params):
        (p * (rank + 1) * (i + 1)).sum().backward()
    assert all(b["launched"] for b in fg._buckets)  # both went out during backward
    fg.finish_exchange()
    for p, e in zip(params, expect):
        assert torch.allclose(p.grad, torch.full_like(p, e)), (rank, p.grad, e)
    fg.zero_()
    (params[2] * 2.0).sum().backward()  # bucket 0 gets nothing on any rank -> skipped, bucket 1 exchanged
    # buckets go out strictly in order: bucket 1 is complete but waits for bucket 0's turn, which comes in finish_exchange
    assert [b["launched"] for b in fg._buckets] == [False, False]
    fg.finish_exchange()
    assert [b["launched"] for b in fg._buckets] == [True, True] and fg._buckets[0]["work"] is None
    assert torch.allclose(params[2].grad, torch.full_like(params[2], 2.0)) and float(params[0].grad.abs().sum()) == 0.0
    from presight_amd.ops import mark_touched
    try:
        mark_touched([params[2]])  # what a HIP backward node does after adding a SECOND contribution in place
        raise SystemExit("a second in-place contribution after the launch must raise")
    except RuntimeError as e:
        assert "second gradient" in str(e)
    # routing left a sub-field without samples on ONE rank only (K > 1): rank 1 never completes bucket 0, rank 0 completes
    # both during backward (bucket 1 first).  Every rank must still issue the collectives in the same order.
    fg.flags_may_differ_across_ranks = True
    fg.zero_()
    (params[2] * (rank + 1.0)).sum().backward()
    (params[0] * (rank + 1.0)).sum().backward()
    if rank == 0:
        (params[1] * 3.0).sum().backward()
    assert [b["launched"] for b in fg._buckets] == ([True, True] if rank == 0 else [False, False])
    fg.finish_exchange()
    assert torch.allclose(params[0].grad, torch.full_like(params[0], 1.5)), params[0].grad
    assert torch.allclose(params[1].grad, torch.full_like(params[1], 1.5)), params[1].grad
    assert torch.allclose(params[2].grad, torch.full_like(params[2], 1.5)), params[2].grad
    assert fg.touched_params() == [0, 1, 2]  # agreed over ranks
    fg.zero_()  # only the agreed touched ranges are cleared
    assert float(fg.flat.abs().sum()) == 0.0
    dist.barrier(); dist.destroy_process_group()
    print("rank", rank, "ok")
""")


_WORKER_SHARDED = textwrap.dedent("""
    import os, sys, torch, torch.distributed as dist
    sys.path.insert(0, {root!r})
    from presight_amd.dist import FlatGrads, init_from_env, intersect_ranges, global_depth_clip
    rank, local, world = init_from_env("cpu")
    torch.manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(5, 3)), torch.nn.Parameter(torch.randn(7)), torch.nn.Parameter(torch.randn(2, 2, 2))]
    fg = FlatGrads(params, bucket_sizes=[2, 1], shard_world=world)
    assert fg.bucket_ranges == [(0, 24), (24, 32)] and fg.total == 32  # every bucket splits into `world` 16-byte aligned shards
    fg.enable_overlap([params[0:2], params[2:3]], mode="sharded")
    # replicated flat parameter buffer (what HipAdam builds) + a plain SGD update on the OWNED shard only
    flat_p = torch.zeros(fg.total)
    for p, off in zip(params, fg.offsets):
        flat_p[off:off + p.numel()] = p.data.reshape(-1)
        p.data = flat_p[off:off + p.numel()].view_as(p)
    before = flat_p.clone()
    for step in range(2):
        fg.zero_()
        for i, p in enumerate(params):
            if step == 1 and i == 2:
                continue  # second step: bucket 1 gets no gradient on any rank
            (p * (rank + 1.0) * (i + 1)).sum().backward()
        fg.finish_exchange()
        owned = fg.owned_ranges()
        assert owned == [(12 * rank, 12 * rank + 12), (24 + 4 * rank, 28 + 4 * rank)], owned
        touched = fg.touched_ranges()
        for a, b in intersect_ranges(touched, owned):
            flat_p[a:b] -= 0.1 * fg.flat[a:b]  # the averaged gradient is only guaranteed inside the owned shard
        fg.gather_params(flat_p, touched)
        fg.wait_params()
    # expected: gradient of parameter i averaged over ranks = 1.5 * (i + 1), two steps for i < 2, one for i = 2
    for i, (p, off) in enumerate(zip(params, fg.offsets)):
        n = p.numel()
        steps = 1 if i == 2 else 2
        assert torch.allclose(flat_p[off:off + n], before[off:off + n] - 0.1 * steps * 1.5 * (i + 1), atol=1e-6), (rank, i)
    # replicas identical
    ref = flat_p.clone(); dist.broadcast(ref, src=0)
    assert torch.equal(ref, flat_p)
    # expected-depth clip bounds over all ranks
    mm = torch.tensor([1.0 + rank, 5.0 - rank])
    global_depth_clip()(mm)
    assert mm.tolist() == [1.0, 5.0]
    dist.barrier(); dist.destroy_process_group()
    print("rank", rank, "ok")
""")


_WORKER_PIECES = textwrap.dedent("""
    import os, sys, torch, torch.distributed as dist
    sys.path.insert(0, {root!r})
    from presight_amd.dist import FlatGrads, init_from_env, intersect_ranges, COMM_LOG
    from presight_amd.ops import mark_touched
    rank, local, world = init_from_env("cpu")
    mode = {mode!r}
    M = (world + 1) / 2.0   # mean over the ranks of (rank + 1)
    torch.manual_seed(0)
    small, table = torch.nn.Parameter(torch.randn(3, 4)), torch.nn.Parameter(torch.randn(32, 2))
    fg = FlatGrads([small, table], bucket_sizes=[1, 1], shard_world=world if mode == "sharded" else 1, splits={{1: 4}})
    t0 = fg.offsets[1]  # (the small bucket is padded to a whole number of shards in sharded mode)
    assert fg.bucket_parts == {{1: [(t0 + 16 * g, t0 + 16 * (g + 1)) for g in range(4)]}}, fg.bucket_parts
    fg.enable_overlap([[small], [table]], mode=mode)
    assert len(fg._buckets) == 5 and table._ps_parts == 4
    flat_p = torch.zeros(fg.total)
    for p, off in zip([small, table], fg.offsets):
        flat_p[off:off + p.numel()] = p.data.reshape(-1)
        p.data = flat_p[off:off + p.numel()].view_as(p)
    before = flat_p.clone()

    def update():
        fg.finish_exchange()
        owned, touched = fg.owned_ranges(), fg.touched_ranges()
        for a, b in intersect_ranges(touched, owned):
            flat_p[a:b] -= 0.1 * fg.flat[a:b]
        fg.gather_params(flat_p, touched)
        fg.wait_params()

    # step 1: a piece-aware producer (field_ops._scatter): MLP-like parameter first, then the table level group by level group
    fg.zero_()
    small.grad.add_(rank + 1.0)
    mark_touched([small])
    assert [b["launched"] for b in fg._buckets] == [True, False, False, False, False]
    for g in range(4):
        table.grad.view(-1)[16 * g:16 * (g + 1)].add_((rank + 1.0) * (g + 1))
        table._ps_part_done(table, g)
        assert [b["launched"] for b in fg._buckets] == [True] + [True] * (g + 1) + [False] * (3 - g)
    mark_touched([table])  # the closing whole-parameter mark of the backward node: nothing left to hand over, no error
    assert all(b["phase"] == "backward" for b in fg._buckets)  # EVERY bucket left before finish_exchange
    update()
    exp = before.clone()
    exp[0:12] -= 0.1 * M
    for g in range(4):
        exp[t0 + 16 * g:t0 + 16 * (g + 1)] -= 0.1 * M * (g + 1)
    assert torch.allclose(flat_p, exp, atol=1e-6), (rank, (flat_p - exp).abs().max())
    # step 2: a producer that does not work in pieces reports the whole parameter: all pieces go out at once, in order
    fg.zero_()
    table.grad.add_(rank + 1.0)
    small.grad.add_(2.0 * (rank + 1.0))
    mark_touched([table])
    assert [b["launched"] for b in fg._buckets] == [False] * 5  # bucket order: the small bucket goes first
    mark_touched([small])
    assert [b["launched"] for b in fg._buckets] == [True] * 5
    update()
    exp[0:12] -= 0.1 * 2.0 * M
    exp[t0:t0 + 64] -= 0.1 * M
    assert torch.allclose(flat_p, exp, atol=1e-6)
    # step 3: the table receives nothing on any rank (off-schedule): its pieces are skipped, only the small bucket is exchanged
    fg.zero_()
    small.grad.add_(rank + 1.0)
    mark_touched([small])
    n_before = COMM_LOG.seq
    update()
    exp[0:12] -= 0.1 * M
    assert torch.allclose(flat_p, exp, atol=1e-6) and COMM_LOG.seq - n_before == (1 if mode == "sharded" else 0)
    # step 4: the FIRST bucket is known to receive nothing on any rank (schedule-driven, e.g. proposal networks off schedule):
    # skip_buckets takes it out of the launch order, the pieces behind it still leave during backward
    fg.zero_()
    fg.skip_buckets([0])
    for g in range(4):
        table.grad.view(-1)[16 * g:16 * (g + 1)].add_(rank + 1.0)
        table._ps_part_done(table, g)
    assert [b["launched"] for b in fg._buckets] == [True] * 5 and [b["phase"] for b in fg._buckets[1:]] == ["backward"] * 4
    mark_touched([table])
    update()
    exp[t0:t0 + 64] -= 0.1 * M
    assert torch.allclose(flat_p, exp, atol=1e-6)
    try:
        fg.zero_()
        fg.skip_buckets([0])
        mark_touched([small])  # a gradient for a bucket that was declared empty
        raise SystemExit("a contribution to a skipped bucket must raise")
    except RuntimeError as e:
        assert "second gradient" in str(e)
    # a piece reported twice is an error
    fg.zero_()
    table._ps_part_done(table, 0)
    try:
        table._ps_part_done(table, 0)
        raise SystemExit("a piece reported twice must raise")
    except RuntimeError as e:
        assert "twice" in str(e)
    for g in range(1, 4):
        table._ps_part_done(table, g)
    mark_touched([small, table])
    fg.finish_exchange()
    ref = flat_p.clone(); dist.broadcast(ref, src=0)
    assert torch.equal(ref, flat_p)
    dist.barrier(); dist.destroy_process_group()
    print("rank", rank, "ok")
""")


@pytest.mark.parametrize("mode,world", [("allreduce", 2), ("sharded", 2), ("sharded", 4)])
def test_split_table_buckets_gloo_world2(tmp_path, mode, world):
    """A hash table exchanged as level-group PIECES (FlatGrads splits): every piece is its own collective, handed over by the producer
    as soon as the accumulate launch of that level group is enqueued -- before backward ends -- strictly in bucket order on every
    rank; a producer that reports the whole parameter, an off-schedule step and the sharded update work as before."""
    script = tmp_path / "worker_pieces.py"
    script.write_text(_WORKER_PIECES.format(root=ROOT, mode=mode))
    port = "29741" if mode == "allreduce" else "29743"
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT=port, PRESIGHT_COMM_LOG=str(tmp_path / "comm_{rank}.log"))
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={world}", "--master-addr", "127.0.0.1",
                        "--master-port", port, str(script)], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert r.stdout.count("ok") == world
    logs = [(tmp_path / f"comm_{r_}.log").read_text().splitlines() for r_ in range(world)]
    assert all(lg == logs[0] for lg in logs)
    kind = "reduce_scatter" if mode == "sharded" else "all_reduce"
    step1 = [ln for ln in logs[0] if f" {kind} " in ln and "step=1" in ln]
    assert len(step1) == 5 and all("phase=backward" in ln for ln in step1)  # all 5 buckets of the first step left during backward
    assert [ln.split("bucket=")[1].split()[0] for ln in step1] == ["0", "1", "2", "3", "4"]


def test_sharded_exchange_gloo_world2(tmp_path):
    """reduce-scatter -> update of the owned shard -> all-gather (presight_amd.dist mode "sharded"): bit-equal replicas"""
    script = tmp_path / "worker_sharded.py"
    script.write_text(_WORKER_SHARDED.format(root=ROOT))
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29733", PRESIGHT_COMM_LOG=str(tmp_path / "comm_{rank}.log"))
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1",
                        "--master-port", "29733", str(script)], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert r.stdout.count("ok") == 2
    # the per-collective sequence log (presight_amd.dist.CommLog): both ranks issued the SAME collectives in the SAME order -- what
    # NCCL / gloo need, and what the next hang will be diagnosed with (first differing / missing line)
    logs = [(tmp_path / f"comm_{r_}.log").read_text().splitlines() for r_ in range(2)]
    assert logs[0] == logs[1] and len(logs[0]) >= 7, logs
    kinds = [ln.split()[1] for ln in logs[0]]
    assert kinds[:2] == ["reduce_scatter", "reduce_scatter"] and kinds.count("all_gather_params") == 3 and "all_reduce_max_depth_clip" in kinds
    assert [int(ln.split()[0]) for ln in logs[0]] == list(range(1, len(logs[0]) + 1))
    assert "bucket=0 bytes=96" in logs[0][0] and "step=1" in logs[0][0]


_WORKER_ONE = textwrap.dedent("""
    import os, sys, torch, torch.distributed as dist
    sys.path.insert(0, {root!r})
    from presight_amd.dist import FlatGrads, init_from_env, exchanging, COMM_LOG
    from presight_amd.ops import mark_touched
    rank, local, world = init_from_env("cpu")
    assert world == 1 and dist.is_initialized() and dist.get_world_size() == 1 and exchanging()
    for mode in ("allreduce", "sharded"):
        torch.manual_seed(0)
        a, b = torch.nn.Parameter(torch.randn(3, 4)), torch.nn.Parameter(torch.randn(32, 2))
        fg = FlatGrads([a, b], bucket_sizes=[1, 1], shard_world=1, splits={{1: 4}})
        fg.enable_overlap([[a], [b]], mode=mode)
        assert not fg.dry and fg._distributed()
        fg.zero_()
        ga, gb = torch.randn(3, 4), torch.randn(32, 2)
        a.grad.add_(ga); mark_touched([a])
        b.grad.add_(gb)
        for g in range(4):
            b._ps_part_done(b, g)
        n0 = COMM_LOG.seq
        assert n0 >= 5 and all(x["launched"] and x["phase"] == "backward" for x in fg._buckets)
        fg.finish_exchange()
        assert torch.equal(a.grad, ga) and torch.equal(b.grad, gb)  # sum over one rank / 1
        assert fg.owned_ranges() == [(0, fg.total)] or mode == "sharded"
        os.environ["PRESIGHT_EXCHANGE_WORLD_OF_ONE"] = "0"
        assert not exchanging() and not fg._distributed()
        os.environ["PRESIGHT_EXCHANGE_WORLD_OF_ONE"] = "1"
    kinds = {{ln.split()[1] for ln in COMM_LOG.tail(64)}}
    assert {{"all_reduce", "reduce_scatter"}} <= kinds, kinds
    dist.destroy_process_group()
    print("ok")
""")


def test_process_group_of_one_exchanges_when_asked(tmp_path):
    """PRESIGHT_EXCHANGE_WORLD_OF_ONE=1: a ONE-rank process group (here gloo; on the GPU box RCCL: test_hip_dist.py) counts as a
    distributed run -- every bucket collective is issued, the result is the identity; without the switch nothing is issued."""
    script = tmp_path / "worker_one.py"
    script.write_text(_WORKER_ONE.format(root=ROOT))
    env = dict(os.environ, RANK="0", LOCAL_RANK="0", WORLD_SIZE="1", MASTER_ADDR="127.0.0.1", MASTER_PORT="29747",
               PRESIGHT_EXCHANGE_WORLD_OF_ONE="1")
    r = subprocess.run([sys.executable, str(script)], capture_output=True, text=True, env=env, timeout=120)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


def test_bench_launcher_and_arguments():
    """bench.py --gpus N outside torchrun starts N ranks itself (before touching the GPU) and refuses a node with fewer GPUs;
    a worker whose WORLD_SIZE disagrees with --gpus fails instead of silently measuring one GPU"""
    import bench

    a = bench.parse_args(["--gpus", "4", "--steps", "3"])
    assert a.gpus == 4 and a.steps == 3 and a.config == "cfg2" and a.scaling is None
    assert bench.CONFIGS["cfg2"]["scaling"] == "weak" and bench.CONFIGS["cfg3"]["scaling"] == "strong"
    env = {k: v for k, v in os.environ.items() if k not in ("WORLD_SIZE", "RANK", "LOCAL_RANK")}
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--gpus", "2", "--steps", "1", "--warmup", "0"], capture_output=True,
                       text=True, env=env, timeout=300)
    assert r.returncode == 2 and "this node has 0 GPU" in r.stderr, (r.returncode, r.stderr[-500:])
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--gpus", "2"], capture_output=True, text=True,
                       env=dict(env, WORLD_SIZE="1", RANK="0", LOCAL_RANK="0"), timeout=300)
    assert r.returncode != 0 and "WORLD_SIZE=1" in (r.stderr + r.stdout)


def test_range_helpers():
    from presight_amd.dist import _merge, intersect_ranges

    assert _merge([(8, 12), (0, 4), (4, 8), (20, 24)]) == [(0, 12), (20, 24)]
    assert intersect_ranges([(0, 10), (20, 30)], [(5, 25)]) == [(5, 10), (20, 25)]
    assert intersect_ranges([(0, 4)], [(4, 8)]) == []


def test_gradient_exchange_gloo_world2(tmp_path):
    script = tmp_path / "worker.py"
    script.write_text(_WORKER.format(root=ROOT))
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29731")
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1",
                        "--master-port", "29731", str(script)], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert r.stdout.count("ok") == 2


def test_flat_grads_touched_ranges():
    """parameters without a gradient in a step are skipped by the optimizer (torch: grad None), adjacent ones merge"""
    from presight_amd.dist import FlatGrads

    ps = [torch.nn.Parameter(torch.randn(n)) for n in (5, 8, 3, 16)]
    fg = FlatGrads(ps)
    assert fg.offsets == [0, 8, 16, 20] and fg.total == 36
    assert fg.touched_ranges() == []
    (ps[0].sum() + ps[1].sum() + ps[3].sum()).backward()
    assert fg.touched() == [True, True, False, True]
    assert fg.touched_ranges() == [(0, 16), (20, 36)]
    ps[2]._ps_touched = True  # what a HIP backward does after writing into the parameter's .grad in place
    assert fg.touched_ranges() == [(0, 36)]
    fg.zero_()
    assert fg.touched_ranges() == [] and float(fg.flat.abs().sum()) == 0.0


def test_lr_schedule_matches_torch_chained_scheduler():
    """WarmupMultiStepSchedule against torch's ChainedScheduler([LinearLR, MultiStepLR]) as built by the reference
    (ns/engine/my_schedulers.py:50-70), scaled-down step counts"""
    from torch.optim import lr_scheduler

    from presight_amd.optim import WarmupMultiStepSchedule

    class _Opt:  # stands in for HipAdam: the schedule only touches .lr
        lr = 1e-2

    max_steps = 400
    ms, warm = [max_steps // 4, max_steps // 2, max_steps * 3 // 4], max_steps // 10
    p = torch.nn.Parameter(torch.zeros(1))
    ref_opt = torch.optim.Adam([p], lr=1e-2)
    ref = lr_scheduler.ChainedScheduler([lr_scheduler.LinearLR(ref_opt, start_factor=0.01, total_iters=warm),
                                         lr_scheduler.MultiStepLR(ref_opt, milestones=ms, gamma=0.33)])
    ours = WarmupMultiStepSchedule(_Opt(), max_steps=max_steps, milestones=ms, warmup_steps=warm)
    for t in range(max_steps):
        assert abs(ours.opt.lr - ref_opt.param_groups[0]["lr"]) <= 1e-9 * 1e-2 + 1e-15, (t, ours.opt.lr, ref_opt.param_groups[0]["lr"])
        ref_opt.step()
        ref.step()
        ours.step()


def test_hip_ops_refuse_cpu_tensors():
    """No CPU fallback: the product path fails loudly when handed CPU tensors."""
    from presight_amd import field_ops, ops

    with pytest.raises(RuntimeError):
        ops.hashgrid_encode(torch.zeros(4, 3), torch.zeros(32, 2), torch.ones(1), 1, 2, 5)
    with pytest.raises(RuntimeError):
        field_ops.field_points(torch.zeros(2, 3), True, pos=torch.zeros(4, 3))


def test_epoch_order_is_the_reference_loader_order():
    """presight_amd.datafeed.epoch_order == iterating torch's DistributedSampler over the reference's ImageChunk
    (ns/data/PreSight/my_datamanager.py:203-212), captured by tests/golden/make_golden.py::gold_datafeed"""
    from presight_amd.datafeed import epoch_order

    G = load_golden("datafeed")
    P = G["rgbs"].shape[0]
    for world, rank in ((1, 0), (3, 1)):
        assert torch.equal(epoch_order(P, world, rank, seed=0), torch.from_numpy(G[f"order_w{world}r{rank}"]))
    # padding by wrap-around keeps every rank's share equal; an unshuffled pass is the identity
    assert epoch_order(10, 4, 3).shape[0] == 3 and epoch_order(10, 1, 0, shuffle=False).tolist() == list(range(10))


def test_lazy_outputs_behave_like_a_dict():
    """presight_amd.model.LazyOutputs: `prop_depth_i` of a training forward is evaluated on first access (the reference renders it
    in every forward, ns/models/PreSight/nerfacto_nusc_ms.py:543-544); membership, order, get / items / values are the plain dict's"""
    from presight_amd.model import LazyOutputs

    calls = []
    o = LazyOutputs({"rgb": 1})
    o.lazy("prop_depth_0", lambda: (calls.append(0), "d0")[1])
    o.lazy("prop_depth_1", lambda: (calls.append(1), "d1")[1])
    assert "prop_depth_0" in o and list(o.keys()) == ["rgb", "prop_depth_0", "prop_depth_1"] and not calls
    assert o["prop_depth_1"] == "d1" and calls == [1] and o["prop_depth_1"] == "d1" and calls == [1]
    assert o.get("prop_depth_0") == "d0" and o.get("missing", 3) == 3 and calls == [1, 0]
    o.lazy("x", lambda: 7)
    assert dict(o.items()) == {"rgb": 1, "prop_depth_0": "d0", "prop_depth_1": "d1", "x": 7} and list(o.values())[-1] == 7
    o.lazy("y", lambda: 8)
    o["y"] = 9  # an explicit assignment wins
    assert o["y"] == 9 and o.pop("x") == 7 and "x" not in o
    # shallow copies go through __getitem__ too (a dict subclass would hand out the None placeholder on CPython's fast paths)
    o.lazy("z", lambda: "dz")
    assert dict(o)["z"] == "dz"
    o.lazy("z2", lambda: "dz2")
    assert {**o}["z2"] == "dz2"
    o.lazy("z3", lambda: "dz3")
    d = {}
    d.update(o)
    assert d["z3"] == "dz3" and o.copy() == d and len(o) == len(d)


def test_bench_line_is_compact():
    """The line of record must survive the driver's bounded stdout tail (round 4 lost its headline to a 29 KB line): `compact_line` of
    the largest committed full record, and of a synthetic worst case (8-GPU run with a long bucket timeline, every secondary shape with
    its dry-run tables, error strings of unbounded length), stays below LINE_BUDGET_BYTES and keeps the contract fields, `roofline` and
    `cpu_baseline`."""
    import bench

    full = json.load(open(os.path.join(ROOT, "profiles", "r04_bench_line_default.json")))
    assert len(json.dumps(full)) > 20000  # (the record that was lost)
    line = bench.compact_line(full, "bench_detail.json")
    text = json.dumps(line, separators=(",", ":"))
    assert len(text) < bench.LINE_BUDGET_BYTES, len(text)
    for k in ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling", "vs_baseline", "dtype",
              "data", "config", "roofline", "cpu_baseline", "end_to_end", "secondary"):
        assert k in line, k
    assert line["value"] == full["value"] and line["ms_per_step"] == full["ms_per_step"]
    assert set(("bound", "achieved", "peak", "unit", "frac", "traffic")) <= set(line["roofline"])
    assert set(("value", "unit", "cores", "kind", "sample")) <= set(line["cpu_baseline"])
    assert "workload" in line["config"] and "model" not in line["config"]
    # worst case: blow every unbounded part up
    worst = json.loads(json.dumps(full))
    worst["n_gpus"] = 8
    tl = [{"bucket": i, "bytes": 671088640, "steps_exchanged": 3, "handed_over_in_backward": 3, "ms_before_backward_end": 1.2345678} for i in range(64)]
    worst["comm"] = {"backend": "nccl", "ranks": 8, "collectives_per_step": 17.0, "gradient_buckets_issued_during_backward_per_step": 7.0,
                     "bytes_on_link_per_rank_per_step": 1.234e9, "bucket_timeline": tl, "exchange_exposed_ms": 1.234,
                     "schedule_by_construction": bench.exchange_schedule(tl, 8, "sharded"), "model": bench.exchange_model(1.234e9, 8)}
    worst["other_scaling"] = dict(scaling="strong", rays_per_gpu=8192, value=1.23456789e7, ms_per_step=5.4321)
    worst["replicas_max_abs_diff"] = 0.0
    for i in range(12):
        worst["secondary"][f"extra_shape_{i}"] = {"error": "RuntimeError: " + "x" * 5000}
    worst["config"]["workload"] = "w" * 5000
    worst["cpu_baseline"]["sample"] = "s" * 5000
    worst["roofline"]["kernel"] = "k" * 5000
    worst["roofline_kernels"] = worst["roofline_kernels"] * 20
    text = json.dumps(bench.compact_line(worst, "bench_detail.json"), separators=(",", ":"))
    assert len(text) < bench.LINE_BUDGET_BYTES + 3000  # emit() drops the optional blocks beyond the budget; the core alone must fit:
    core = bench.compact_line(worst, "bench_detail.json")
    for k in ("secondary", "comm", "other_scaling", "psnr_after_k_steps", "psnr_vs_oracle"):
        core.pop(k, None)
    assert len(json.dumps(core, separators=(",", ":"))) < bench.LINE_BUDGET_BYTES
    # emit(): last stdout line parses, is compact, and the detail file holds the full record
    import contextlib
    import io
    import tempfile

    with tempfile.TemporaryDirectory() as td:
        old = bench.DETAIL_FILE
        bench.DETAIL_FILE = os.path.join(td, "detail.json")
        try:
            buf = io.StringIO()
            with contextlib.redirect_stdout(buf):
                bench.emit(worst)
            last = buf.getvalue().strip().splitlines()[-1]
            assert len(last) < bench.LINE_BUDGET_BYTES
            got = json.loads(last)
            assert got["value"] == worst["value"] and "roofline" in got and "cpu_baseline" in got
            assert json.load(open(bench.DETAIL_FILE))["roofline_kernels"] == worst["roofline_kernels"]
        finally:
            bench.DETAIL_FILE = old


def test_trainer_notices_a_sub_module_left_in_eval_mode():
    """the per-step fast path (skip nn.Module.train()'s walk over ~1000 modules) must not let a sub-module that somebody put
    into eval mode on its own stay there: the check reads the flags three levels deep (model -> field / samplers -> sub-fields)"""
    from presight_amd.trainer import _some_module_in_eval_mode

    class Leaf(torch.nn.Module):
        pass

    class Mid(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.fields = torch.nn.ModuleList([Leaf(), Leaf()])

    class Top(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.field, self.sampler = Mid(), Leaf()

    m = Top().train()
    assert not _some_module_in_eval_mode(m)
    m.sampler.eval()
    assert m.training and _some_module_in_eval_mode(m)
    m.train()
    m.field.fields[1].eval()  # depth 3: top -> field -> fields (ModuleList) -> sub-field
    assert _some_module_in_eval_mode(m)
    m.train()
    assert not _some_module_in_eval_mode(m)


_WORKER_SPARSE = textwrap.dedent("""
    import os, sys, torch, torch.distributed as dist
    sys.path.insert(0, {root!r})
    from presight_amd.dist import FlatGrads, init_from_env, intersect_ranges, COMM_LOG
    from presight_amd.ops import mark_touched
    rank, local, world = init_from_env("cpu")
    torch.manual_seed(0)
    K, L, LS, F = 1, 2, 2, 1                      # 2 levels x 4 slices of 4 rows: 8 items, 32 table entries
    n_slices, rows = 4, 1 << LS
    n_items = K * L * n_slices
    small, table = torch.nn.Parameter(torch.randn(3, 4)), torch.nn.Parameter(torch.randn(n_items * rows, F))

    def build(sparse):
        for p in (small, table):
            for a in ("_ps_sparse", "_ps_bucket", "_ps_on_touch", "_ps_parts", "_ps_part_done", "_ps_part_buckets"):
                if hasattr(p, a):
                    delattr(p, a)
        fg = FlatGrads([small, table], bucket_sizes=[1, 1], shard_world=world)
        fg.enable_overlap([[small], [table]], mode="sharded", sparse=[1] if sparse else [])
        return fg

    # this rank's records: item i holds n_i = (i + rank) % 3 + (i == 5) * 6 records, its stream is sized for an UPPER bound of them
    g = torch.Generator().manual_seed(100 + rank)
    n = [(i + rank) % 3 + (6 if i == 5 else 0) for i in range(n_items)]
    upper = [c + (i + 2 * rank) % 3 for i, c in enumerate(n)]
    starts, off = [], 0
    for u in upper:
        starts.append(off)
        off += (u + 3) // 4 * 4
    n_rec_max = off + 8
    rec_idx = torch.full((n_rec_max,), -1, dtype=torch.int32)
    rec_val = torch.full((F + 1, n_rec_max), float("nan"))
    dense = torch.zeros(n_items * rows)             # what the plain (dense) table backward of this rank would have written
    for i in range(n_items):
        for j in range(n[i]):
            row, val = int(torch.randint(0, rows, (1,), generator=g)), float(torch.randint(-8, 9, (1,), generator=g))
            rec_idx[starts[i] + j] = row | (31 << 16)                       # t = 31: a single corner, weight already applied
            rec_val[0, starts[i] + j], rec_val[F, starts[i] + j] = val, 0.0
            dense[i * rows + row] += val
    lay = [0, 4096, 4096 + 4 * n_items, 4096 + 8 * n_items, 4096 + 8 * n_items + 4 * ((n_items + 3) // 4 * 4), 0, n_rec_max, n_items, LS]
    lay[5] = lay[4] + 4 * n_rec_max
    ws = torch.zeros(lay[5] + 4 * (F + 1) * n_rec_max, dtype=torch.uint8)
    put = lambda o, t: ws[o:o + t.numel() * 4].copy_(t.contiguous().view(torch.uint8).reshape(-1))
    gmax = torch.tensor([1.0 + rank, 4.0 - rank]).view(torch.int32)          # per-level maxima differ between the ranks
    put(lay[0], gmax)
    put(lay[1], torch.tensor([s + c for s, c in zip(starts, n)], dtype=torch.int32))   # cursors = stream ends
    put(lay[2], torch.tensor(upper, dtype=torch.int32))
    put(lay[3], torch.tensor(starts, dtype=torch.int32))
    put(lay[4], rec_idx)
    put(lay[5], rec_val)
    seen = {{}}

    def make_accumulate(fg):
        def accumulate(run_starts, run_counts, n_runs, ridx, rval, stride, gmax_bits, n_points_total, out_scale, i0, i1):
            # the owner's pass: every run of every owned item, summed exactly (small integers), scaled, WRITTEN into its shard
            seen.update(gmax=gmax_bits.view(torch.float32).tolist(), n_total=n_points_total, n_runs=n_runs)
            out = fg.flat[fg.offsets[1]:fg.offsets[1] + n_items * rows]
            for li in range(i1 - i0):
                acc = torch.zeros(rows, dtype=torch.float64)
                for r in range(n_runs):
                    b, c = int(run_starts[r, li]), int(run_counts[r, li])
                    assert b % 4 == 0
                    for j in range(c):
                        assert int(ridx[b + j]) >> 16 == 31 and rval[F, b + j] == 0.0
                        acc[int(ridx[b + j]) & 0xffff] += float(rval[0, b + j])
                out[(i0 + li) * rows:(i0 + li + 1) * rows] = (acc * out_scale).float()
        return accumulate

    flat_p = {{}}
    for mode in ("dense", "sparse"):
        fg = build(mode == "sparse")
        fp = torch.zeros(fg.total)
        for p, o in zip([small, table], fg.offsets):
            fp[o:o + p.numel()] = torch.arange(p.numel(), dtype=torch.float32)
        fg.zero_()
        small.grad.add_(rank + 1.0)
        mark_touched([small])
        if mode == "sparse":
            fg.sparse_records(1, dict(ws=ws, layout=lay, L=L, F=F, log2T=4, K=K, n_points=1000 + 24 * rank, accumulate=make_accumulate(fg)))
        else:
            table.grad.view(-1).add_(dense)
        mark_touched([table])
        assert all(b["launched"] and b["phase"] == "backward" for b in fg._buckets)   # both buckets left during "backward"
        fg.finish_exchange()
        owned, touched = fg.owned_ranges(), fg.touched_ranges()
        t0 = fg.offsets[1]
        half = n_items * rows // world
        assert (t0 + rank * half, t0 + (rank + 1) * half) in [(max(a, t0), b) for a, b in owned if b > t0]      # the r-th half of the table
        for a, b in intersect_ranges(touched, owned):
            fp[a:b] -= 0.25 * fg.flat[a:b]
        fg.gather_params(fp, touched)
        fg.wait_params()
        ref = fp.clone(); dist.broadcast(ref, src=0)
        assert torch.equal(ref, fp), mode                                                                         # replicas bit-identical
        flat_p[mode] = fp
    assert torch.equal(flat_p["dense"], flat_p["sparse"])   # integer-valued gradients: the record exchange IS the dense sharded result
    both = [torch.zeros_like(dense) for _ in range(world)]
    dist.all_gather(both, dense)
    exp = torch.arange(n_items * rows, dtype=torch.float32) - 0.25 * sum(both) / world
    assert torch.equal(flat_p["sparse"][t0:t0 + n_items * rows], exp)
    assert seen["gmax"] == [float(world), 4.0] and seen["n_total"] == (1000 + 24 * (world - 1)) * world and seen["n_runs"] == world  # MAX over the ranks of both
    kinds = [ln.split()[1] for ln in COMM_LOG.tail(64)]
    assert kinds.count("all_to_all_records") == F + 2 and "all_reduce_max_levels" in kinds and "all_to_all_item_runs" in kinds
    dist.barrier(); dist.destroy_process_group()
    print("rank", rank, "ok")
""")


@pytest.mark.parametrize("world", [2, 4])
def test_sparse_record_exchange_gloo_world2(tmp_path, world):
    """exchange = sparse: a hash table's gradient travels as the binned backward's RECORD streams to the owners of its
    slices (all_to_all of the streams + per-item run tables, per-level maxima MAX-reduced first), the owner accumulates every rank's run
    and writes its shard of the mean; Adam-on-the-shard and the parameter all-gather are the sharded mode's.  Two / four gloo ranks on the CPU
    with a stand-in accumulate pass: replicas bit-identical, and -- on integer-valued records, where float sums are exact -- bit-equal
    to the DENSE sharded exchange of the same gradients; streams sized for upper bounds, empty runs and a hot slice included."""
    script = tmp_path / "worker_sparse.py"
    script.write_text(_WORKER_SPARSE.format(root=ROOT))
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29747")
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={world}", "--master-addr", "127.0.0.1",
                        "--master-port", "29747", str(script)], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
    assert r.stdout.count("ok") == world


def test_traffic_of_launches_over_parts_is_refused(tmp_path):
    """tools/pmc_traffic.py averages a counter over a kernel's launches: a summary in which the accumulation was launched over parts of the table
    as well (more launches than the binning had) gives no figure"""
    def summary(added):
        lines = ["src_sha16=0123456789abcdef"]
        for counter in ("FETCH_SIZE", "WRITE_SIZE"):
            lines.append(f"== pass: --pmc {counter} (rc=0)")
            for name, launches, avg in (("main_fwd_kernel", 31, 10.0), ("bin_kernel<2, false, 3>", 31, 20.0), ("accumulate_kernel<2>", added, 30.0)):
                lines += [f"void (anonymous namespace)::{name}(float const*, floa", f"    {counter:36s} launches {launches:4d}  avg {avg:18.1f}"]
        path = tmp_path / f"summary_{added}.txt"
        path.write_text("\n".join(lines) + "\n")
        return path

    out = tmp_path / "traffic.json"
    run = lambda path: subprocess.run([sys.executable, os.path.join(ROOT, "tools", "pmc_traffic.py"), str(path), str(out)],  # noqa: E731
                                      capture_output=True, text=True, timeout=120)
    r = run(summary(55))
    assert r.returncode != 0 and "part of the table" in r.stderr and not out.exists()
    r = run(summary(31))
    assert r.returncode == 0, r.stderr[-500:]
    got = json.loads(out.read_text())
    assert got["kernels"]["accumulate_kernel"]["hbm_bytes_per_launch"] == (2 * 30 + 30) * 1024
