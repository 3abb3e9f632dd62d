"""CPU-only: options of scripts/train.py that contradict each other end in an error, before anything runs."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def cli():
    spec = importlib.util.spec_from_file_location('w2s_train_cli_mixer', os.path.join(ROOT, 'scripts', 'train.py'))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_a_mixer_for_the_model_without_one(tmp_path, capsys):
    with pytest.raises(SystemExit):
        cli().main(['--model', 'ppgnet', '--signals', 'PPG', '--sequence-mixer', 'ssm', '--out', str(tmp_path)])
    assert '--sequence-mixer' in capsys.readouterr().err
