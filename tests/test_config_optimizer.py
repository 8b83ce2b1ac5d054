"""The optimizer block of an experiment file: what Adam ignores, and what AdamW wants."""
import os

import pytest
import yaml


@pytest.fixture
def load(golden_dir, tmp_path):
    from nerf_kinematics_amd import config as config_mod
    with open(os.path.join(golden_dir, "lego-lowres3_config.yml")) as fh:
        cfg = yaml.safe_load(fh)

    def load(**opt):
        path = tmp_path / "c.yml"
        path.write_text(yaml.safe_dump(dict(cfg, optimizer=dict(cfg["optimizer"], **opt))))
        return config_mod.load_config(str(path))
    return load


@pytest.mark.parametrize("more", [dict(weight_decay=None), dict(weight_decay="none"), dict(state_bits=None), dict(state_bits="fp32"), dict(weight_decay=[0.1])])
def test_adam_ignores_the_keys_of_adamw(load, more):
    """Files written for Adam may hold anything under keys that Adam does not read."""
    from nerf_kinematics_amd.trainer import TrainOpts
    for kind in (dict(), dict(type="Adam")):
        o, plain = TrainOpts.from_config(load(**kind, **more)), TrainOpts.from_config(load(**kind))
        assert o == plain and o.optimizer == "Adam"


@pytest.mark.parametrize("bad", [dict(weight_decay=None), dict(weight_decay="none"), dict(weight_decay=float("nan")), dict(weight_decay=float("inf")), dict(weight_decay=[0.1]),
                                 dict(state_bits=None), dict(state_bits="fp32"), dict(state_bits=8.5)])
def test_adamw_names_the_key_that_it_cannot_use(load, bad):
    from nerf_kinematics_amd import config as config_mod
    with pytest.raises(config_mod.ConfigError, match="optimizer." + list(bad)[0]):
        load(type="AdamW", **bad)
