"""evaluate / evaluateSingleNode -- the reference's alegnn/modules/evaluation.py:18-168; predictTop: a classifier's answers in full.

Test-set cost of the 'Best' and the 'Last' checkpoint; returns {'costBest', 'costLast'} and (doSaveVars) pickles it to
<saveDir>/evalVars/<name>evalVars.pkl.  Under torch.distributed every rank evaluates its identical replica; rank 0 writes.
"""
from __future__ import annotations

import os
import pickle

import torch
import torch.distributed as dist

from ..functional_out import token_log_probs


def _run(model, data, forward, kwargs):
    doSaveVars = kwargs.get('doSaveVars', True)
    xTest, yTest = data.getSamples('test')
    xTest = xTest.to(model.device)
    yTest = yTest.to(model.device)
    evalVars = {}
    for label in ('Best', 'Last'):                                  # evaluation.py:58-71
        model.load(label=label)
        with torch.no_grad():
            evalVars['cost' + label] = float(data.evaluate(forward(xTest), yTest))
    rank = dist.get_rank() if dist.is_available() and dist.is_initialized() else 0
    if doSaveVars and rank == 0:
        saveDirVars = os.path.join(model.saveDir, 'evalVars')
        os.makedirs(saveDirVars, exist_ok=True)
        with open(os.path.join(saveDirVars, model.name + 'evalVars.pkl'), 'wb') as f:
            pickle.dump(evalVars, f)
    return evalVars


def evaluate(model, data, **kwargs):
    return _run(model, data, lambda x: model.archit(x), kwargs)


def evaluateSingleNode(model, data, **kwargs):
    assert 'singleNodeForward' in dir(model.archit)                 # evaluation.py:109-110
    assert 'getLabelID' in dir(data)
    targetIDs = data.getLabelID('test')
    return _run(model, data, lambda x: model.archit.singleNodeForward(x, targetIDs), kwargs)


def predictTop(model, data, samplesType='test', top=5, temperature=1.0, batchSize=None):
    """What the model's architecture, as it stands, answers on a split of a classification data set (outputs B x classes [x nodes], labels B [x nodes]):
    a dict of 'logProb' [B] (of the true class), 'entropy' [B], and the `top` best classes per sample 'topLogProb' / 'topClasses' [B, top], under
    softmax(output / temperature).  (topClasses, topLogProb) of the training split is what Trainer takes as teacherTop."""
    x, y = data.getSamples(samplesType)
    n = x.shape[0]
    assert n > 0 and (batchSize is None or batchSize > 0)
    step = n if batchSize is None else int(batchSize)
    parts = []
    with torch.no_grad():
        for b in range(0, n, step):
            out = model.archit(x[b:b + step].to(model.device))
            labels = y[b:b + step].to(model.device).to(torch.int64).reshape(out.shape[:1] + out.shape[2:])
            parts.append(token_log_probs(out, labels, top=min(int(top), out.shape[1]), temperature=temperature, dim=1))
    names = ('logProb', 'entropy', 'topLogProb', 'topClasses')
    return {k: None if parts[0][i] is None else torch.cat([p[i] for p in parts]) for i, k in enumerate(names)}
