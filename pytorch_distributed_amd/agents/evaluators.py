"""Evaluator process: every `evaluator_freq` seconds pull a weight snapshot,
play `evaluator_nepisodes` greedy episodes in an eval-mode env, publish the
totals for the logger, and write the checkpoint -- the only checkpoint writer,
as in the reference (core/single_processes/evaluators.py:9-102).
"""
import time

import torch

from ..ops.scan import linear_scan
from ..utils.checkpoint import save_state_dict
from ..utils.helpers import reset_experience
from ..utils.param_store import sync_params


def run_episodes(env, model, nepisodes, early_stop, device=torch.device("cpu"), verbose=None, trace=None):
    """Greedy rollouts; returns (total_steps, total_reward, nepisodes, nepisodes_solved).  trace: a list that receives
    (reward, episode ended, value the model gave the state) per step."""
    experience = reset_experience()
    episode_steps, episode_reward = 0, 0.0
    total_steps, total_reward, done_eps, solved = 0, 0.0, 0, 0
    flag_reset = True
    while done_eps < nepisodes:
        if flag_reset:
            episode_steps, episode_reward = 0, 0.0
            experience = env.reset()
            assert experience.state1 is not None
            flag_reset = False
        action, _, value = model.get_action(experience.state1, device=device)
        experience = env.step(action)
        if experience.terminal1:
            solved += 1
            flag_reset = True
        if early_stop and (episode_steps + 1) >= early_stop:
            flag_reset = True
        episode_steps += 1
        episode_reward += experience.reward
        if trace is not None:
            trace.append((float(experience.reward), flag_reset, float(value)))
        if flag_reset:
            done_eps += 1
            total_steps += episode_steps
            total_reward += episode_reward
            if verbose:
                print(verbose, done_eps)
    return total_steps, total_reward, done_eps, solved


@torch.no_grad()
def returns_report(trace, gamma, device=torch.device("cpu")):
    """-> (mean discounted return of the trace's episodes, mean over its steps of the model's value minus the return that
    followed): G_t = r_t + gamma G_{t+1} as ONE reversed linear recurrence, an episode per row (so that the CPU path, which goes
    step by step, takes the longest episode's steps and not all of them).  An episode that was cut short counts as ended there."""
    if not trace:
        return 0.0, 0.0
    ends = [i + 1 for i, (_, end, _) in enumerate(trace) if end]
    if not ends or ends[-1] != len(trace):
        ends.append(len(trace))
    n = torch.tensor([end - start for start, end in zip([0] + ends, ends)])
    live = torch.arange(int(n.max()))[None, :] < n[:, None]
    rewards = torch.zeros(live.shape)
    rewards[live] = torch.tensor([r for r, _, _ in trace], dtype=torch.float32)
    rewards, n, live = rewards.to(device), n.to(device), live.to(device)
    returns, _ = linear_scan(rewards, torch.full_like(rewards, float(gamma)), reverse=True, lengths=n)
    values = torch.tensor([v for _, _, v in trace], dtype=torch.float32).to(device)
    return float(returns[:, 0].mean()), float((values - returns[live]).mean())


def evaluator(process_ind, args, global_logs, evaluator_logs, env_prototype, model_prototype, global_model):
    print("---------------------------->", process_ind, "evaluator")
    ap = args.agent_params
    env = env_prototype(args.env_params, process_ind)
    env.eval()
    local_device = torch.device(getattr(args, "actor_device", "cpu"))
    local_model = model_prototype(args.model_params, args.norm_val, args.state_shape,
                                  args.action_space, args.action_shape).to(local_device)
    sync_params(local_model, global_model)
    local_model.eval()
    torch.set_grad_enabled(False)
    torch.set_num_threads(max(1, min(2, torch.get_num_threads())))     # the env workers need the cores
    poll = float(getattr(ap, "poll_interval", 5.0))

    def evaluate_and_save():
        sync_params(local_model, global_model)
        trace = [] if getattr(ap, "evaluate_returns", False) else None
        total_steps, total_reward, nepisodes, solved = run_episodes(
            env, local_model, ap.evaluator_nepisodes, args.env_params.early_stop, local_device, trace=trace)
        if trace is not None:
            ret, bias = returns_report(trace, ap.gamma, torch.device(getattr(args, "device", "cpu")))
        with evaluator_logs.logger_lock.get_lock():
            evaluator_logs.total_steps.value = total_steps
            evaluator_logs.total_reward.value = total_reward
            evaluator_logs.nepisodes.value = nepisodes
            evaluator_logs.nepisodes_solved.value = solved
            if trace is not None:
                evaluator_logs.discounted_return.value, evaluator_logs.value_bias.value = ret, bias
            evaluator_logs.logger_lock.value = True
        print("Saving model " + args.model_name + " ...")
        save_state_dict(local_model, args.model_name)
        print("Saved  model " + args.model_name + ".")
        # optional "solved": end the job once an evaluation reaches the target score (bench/pong_wallclock.py measures
        # the wall-clock to that point; the reference only ever stops at `steps`)
        goal = getattr(ap, "stop_at_eval_reward", None)
        if goal is not None and nepisodes > 0 and total_reward / nepisodes >= float(goal):
            print("[evaluator] avg reward %.2f >= %.2f: stopping the job" % (total_reward / nepisodes, float(goal)), flush=True)
            global_logs.stop.value = True

    last_eval_time = time.time()
    while global_logs.running(ap.steps):
        time.sleep(poll)
        if time.time() - last_eval_time > ap.evaluator_freq:
            evaluate_and_save()
            last_eval_time = time.time()
    if not global_logs.stop.value:
        evaluate_and_save()     # final weights always get evaluated and checkpointed
